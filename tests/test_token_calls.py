"""What the operators on rows of tokens refuse, and that a refused call enqueues nothing: seen on the CPU, where nothing runs."""
import pytest

from launch_recorder import recorded  # noqa: F401

SETUP = """
from nvshmem_amd import Runtime
from nvshmem_amd.host import NvshmemError
rt = Runtime(npes=4, symmetric_size=8 << 20)
room = rt.malloc(4 << 20)
A = [room + i * (64 << 10) for i in range(48)]     # operands of up to 64 KiB, apart from each other
END = room + rt.ptr(room, 1) - rt.ptr(room, 0) - 2048      # of what PE 0 may use
launches()

def refused(call, *args, text="", **named):
    try:
        call(*args, **named)
    except NvshmemError as e:
        assert text in str(e), str(e)
    else:
        raise AssertionError("not refused: %s %r" % (call.__name__, args))
    assert not launches()

def taken(call, *args, **named):
    call(*args, **named)
    return [l[0] for l in launches()]
"""

EMBEDDING = SETUP + """
T, V, D = 10, 23, 40
good = ("float", A[0], A[1], A[2], T, V, D)
assert len(taken(rt.embedding, *good)) == 1
def at(i, value, call=rt.embedding, base=good, **more):
    args = list(base)
    args[i] = value
    refused(call, *args, **more)
for i, name in ((1, "out"), (2, "table"), (3, "ids")):
    at(i, None, text="embedding %s" % name)
    at(i, 0x1234, text="not a symmetric address")
    at(i, END - 64, text="leave")
    at(i, A[i - 1] + 2, text="aligned")
at(1, A[1] + 4, text="overlaps")
at(1, rt.ptr(A[1], 2), text="overlaps")                # the same object, named by another PE's copy
at(4, 1 << 40, text="tokens")
at(4, 1 << 63, text="tokens")
at(5, 0, text="rows")
at(5, 1 << 31, text="rows")
at(5, 1 << 20, text="leave")
at(6, 0, text="elements")
at(6, (1 << 24) + 1, text="elements")
refused(rt.embedding, *good, scale=float("nan"), text="scale")
refused(rt.embedding, *good, scale=float("inf"), text="scale")
assert len(taken(rt.embedding, "half", A[0] + 2, A[1] + 6, A[2], T, V, D)) == 1     # any element of a buffer
assert taken(rt.embedding, "half", None, A[1], None, 0, V, D) == []
grad = ("bfloat16", A[0], A[1], A[2], A[3], T, V, D)
assert taken(rt.embedding_grad, *grad)
for i, name in ((1, "dtable"), (2, "dout"), (3, "ids"), (4, "workspace")):
    at(i, None, rt.embedding_grad, grad, text="embedding_grad %s" % name)
    at(i, 0x1234, rt.embedding_grad, grad, text="not a symmetric address")
    at(i, A[i - 1] + 1, rt.embedding_grad, grad, text="aligned")
at(4, A[3] + 32, rt.embedding_grad, grad, text="aligned")
at(4, A[1], rt.embedding_grad, grad, text="overlaps")
at(4, A[0], rt.embedding_grad, grad, text="overlaps")
at(1, A[1], rt.embedding_grad, grad, text="overlaps")
at(5, 1 << 30, rt.embedding_grad, grad)
need = rt.workspace_bytes("embedding_grad", T, V, D)
assert need > 0
at(4, END - need // 64 * 64 + 64, rt.embedding_grad, grad, text="leave")
"""

ROUTER = SETUP + """
T, E, K = 10, 64, 4
good = ("float", A[0], A[1], A[2], A[3], A[4], T, E, K)
names = ("expert", "gate", "counts", "workspace", "logits")
def at(i, value, call, base, **more):
    args = list(base)
    args[i] = value
    refused(call, *args, **more)
assert taken(rt.moe_route, *good) and taken(rt.moe_route, *good, loss=A[5], balance=A[6])
for i, name in enumerate(names, 1):
    at(i, None, rt.moe_route, good, text="moe_route %s" % name)
    at(i, 0x1234, rt.moe_route, good, text="not a symmetric address")
    at(i, A[i - 1] + 2, rt.moe_route, good, text="aligned")
    if name != "logits":
        at(i, A[4], rt.moe_route, good, text="overlaps")
at(2, A[0], rt.moe_route, good, text="overlaps")
refused(rt.moe_route, *good, loss=A[5], text="together")
refused(rt.moe_route, *good, balance=A[5], text="together")
refused(rt.moe_route, *good, loss=A[5], balance=A[5], text="overlaps")
refused(rt.moe_route, *good, loss=A[5], balance=A[4], text="overlaps")
for experts, topk in ((0, 1), (1025, 4), (64, 0), (64, 17), (3, 4), (-5, 1), (64, -1)):
    refused(rt.moe_route, *good[:7], experts, topk)
    refused(rt.moe_route_grad, "float", A[0], A[1], A[2], A[3], T, experts, topk)
    refused(rt.moe_place, A[0], A[1], A[2], A[3], A[4], A[5], A[6], T, topk, experts, 100)
at(6, 1 << 31, rt.moe_route, good, text="tokens")
at(6, 1 << 62, rt.moe_route, good, text="tokens")
at(6, 1 << 18, rt.moe_route, good, text="leave")
refused(rt.moe_route, *good, scale=float("nan"), text="scale")
assert taken(rt.moe_route, "half", None, None, A[2], A[3], None, 0, E, K, loss=A[5], balance=A[6])   # counts are zeros

grad = ("half", A[0], A[1], A[2], A[3], T, E, K)
assert len(taken(rt.moe_route_grad, *grad)) == 1
for i, name in enumerate(("dlogits", "logits", "expert", "dgate"), 1):
    at(i, None, rt.moe_route_grad, grad, text="moe_route_grad %s" % name)
    at(i, A[i - 1] + 1, rt.moe_route_grad, grad, text="aligned")
at(1, A[1], rt.moe_route_grad, grad, text="overlaps")
refused(rt.moe_route_grad, *grad, balance=A[5], text="together")
refused(rt.moe_route_grad, *grad, dloss=A[5], text="together")
refused(rt.moe_route_grad, *grad, balance=A[5], dloss=A[0], text="overlaps")
refused(rt.moe_route_grad, *grad, scale=float("inf"), text="scale")
assert taken(rt.moe_route_grad, "half", None, None, None, None, 0, E, K) == []

place = (A[0], A[1], A[2], A[3], A[4], A[5], A[6], T, K, E, 100)
assert len(taken(rt.moe_place, *place)) == 1
for i, name in ((0, "dest_pe"), (1, "dest_row"), (2, "expected"), (3, "expert_row"), (5, "expert"), (6, "counts")):
    at(i, None, rt.moe_place, place, text="moe_place %s" % name)
    at(i, A[i] + 2, rt.moe_place, place, text="aligned")
at(0, A[5], rt.moe_place, place, text="overlaps")
at(1, A[0], rt.moe_place, place, text="overlaps")
at(9, 62, rt.moe_place, place, text="same number")
many = (A[0], A[8], A[2], A[3], A[4], A[20], A[6], 3000, K, E, 100)     # of many copies: through the workspace
assert taken(rt.moe_place, *many)
"""

COMBINE = SETUP + """
T, K, D, CAP = 10, 3, 40, 50
good = ("float", A[0], A[1], CAP, A[2], A[3], A[4], T, K, D)
def at(i, value, call=rt.moe_combine_sum, base=good, **more):
    args = list(base)
    args[i] = value
    refused(call, *args, **more)
assert len(taken(rt.moe_combine_sum, *good)) == 1
for i, name in ((1, "out"), (2, "recv"), (4, "gate"), (5, "dest_pe"), (6, "dest_row")):
    if name != "gate":
        at(i, None, text="moe_combine_sum %s" % name)
    at(i, 0x1234, text="not a symmetric address")
    at(i, A[6] + 2, text="aligned")
assert len(taken(rt.moe_combine_sum, *good[:4], None, *good[5:])) == 1
at(1, A[1], text="overlaps")
at(1, A[1] + CAP * D * 4 - 4, text="overlaps")
at(1, A[2], text="overlaps")
at(3, 1 << 40, text="leave")
at(7, 1 << 31, text="tokens")
at(8, 0, text="copies")
at(8, 1025, text="copies")
at(9, 0, text="elements")
at(9, 1 << 25, text="elements")
grad = ("half", A[0], A[1], A[2], A[3], CAP, A[4], A[5], A[6], T, K, D)
assert len(taken(rt.moe_combine_grad, *grad)) == 1
for i, name in ((1, "drecv"), (2, "dgate"), (3, "dout"), (4, "recv"), (6, "gate"), (7, "dest_pe"), (8, "dest_row")):
    at(i, None, rt.moe_combine_grad, grad, text="moe_combine_grad %s" % name)
    at(i, A[8] + 1, rt.moe_combine_grad, grad, text="aligned")
assert len(taken(rt.moe_combine_grad, "half", A[3], *grad[2:])) == 1                     # in place
at(1, A[3] + 2, rt.moe_combine_grad, grad, text="overlaps")
at(1, A[2], rt.moe_combine_grad, grad, text="overlaps")
at(2, A[4], rt.moe_combine_grad, grad, text="overlaps")
at(2, A[3], rt.moe_combine_grad, grad, text="overlaps")
at(3, A[0], rt.moe_combine_grad, grad, text="overlaps")
at(5, 1 << 62, rt.moe_combine_grad, grad, text="leave")
"""


@pytest.mark.parametrize("code", [EMBEDDING, ROUTER, COMBINE], ids=["embedding", "router", "combine"])
def test_refusals(recorded, code):  # noqa: F811
    recorded(code)


def test_before_init(recorded):  # noqa: F811
    recorded("""
for t in ("float", "half", "bfloat16"):
    assert getattr(lib, "nvshmemx_amd_%s_embedding_on_stream" % t)(1, 1, 1, 1, 1, 1, 1.0, None) != 0
    assert b"before nvshmem_init" in lib.nvshmemx_amd_last_error()
assert lib.nvshmemx_amd_moe_place_on_stream(1, 1, 1, 1, 1, 1, 1, 1, 1, 8, 1, None) != 0
assert lib.nvshmemx_amd_embedding_grad_workspace(10, 10, 10) == 0
assert lib.nvshmemx_amd_moe_route_workspace(10, 10) == 0
assert lib.nvshmemx_amd_moe_place_workspace(10, 1, 10) == 0
assert not launches()
""")


def test_no_grid_leaves_its_limits(recorded):  # noqa: F811
    """A launch holds fewer than 2^32 threads, in at most 65535 blocks along y and z (the recorder refuses others)."""
    recorded("""
from nvshmem_amd import Runtime
rt = Runtime(npes=4, symmetric_size=40 << 30)
p = [rt.malloc(4 << 30) for _ in range(9)]
launches()
T = (1 << 29) - 8
rt.embedding("half", p[0], p[1], p[2], T, 5, 1)
rt.embedding("half", p[0], p[1], p[2], 60, 5, 1 << 24)
rt.embedding_grad("float", p[0], p[1], p[2], p[3], 9, 5, 1 << 24)
rt.moe_combine_sum("float", p[0], p[1], 3, None, p[2], p[3], 9, 1, 1 << 24)
rt.moe_combine_grad("float", p[0], p[4], p[1], p[5], 3, p[6], p[2], p[3], 9, 1, 1 << 24)
rt.moe_combine_sum("half", p[0], p[1], 10, None, p[2], p[3], T, 1, 1)
rt.moe_combine_grad("half", p[0], p[4], p[1], p[5], 10, p[6], p[2], p[3], T, 1, 1)
rt.moe_route("half", p[0], p[1], p[2], p[3], p[4], 1 << 27, 4, 1, loss=p[5], balance=p[6])
rt.moe_route_grad("half", p[0], p[1], p[2], p[3], 1 << 27, 4, 1)
rt.moe_place(p[0], p[1], p[2], p[3], p[4], p[5], p[6], 1 << 29 - 1, 1, 4, 1 << 40)
rt.embedding_grad("half", p[0], p[1], p[2], p[3], 1 << 24, 1 << 30, 1)
rt.embedding_grad("half", p[0], p[1], p[2], p[3], 1 << 24, (1 << 31) - 1, 1)
assert len(launches()) > 15
""")


WORKSPACES = """
import itertools
from nvshmem_amd import Runtime
rt = Runtime(npes=%d, symmetric_size=1 << 20)

def never_falls(op, *grids):
    size = {p: rt.workspace_bytes(op, *p) for p in itertools.product(*grids)}
    for p, n in size.items():
        for i, grid in enumerate(grids):
            at = grid.index(p[i])
            q = p[:i] + (grid[max(at - 1, 0)],) + p[i + 1:]
            assert 0 <= size[q] <= n, "%%s of %%r takes %%d bytes, of %%r %%d" %% (op, q, size[q], p, n)

def around(*values):
    return sorted({v + d for v in values for d in (-1, 0, 1) if v + d >= 0})

tokens = around(0, 2, 16, 64, 100, 128, 151, 329, 1024, 1207, 2048, 4096, 8192, 16129, 16384, 20000, 65536, 131072, 1 << 20,
                1 << 22, (1 << 31) // rt.npes // 16 - 1)
experts = around(2, 8, 64, 176, 256, 512, 1023)
never_falls("moe_route", tokens, experts)
never_falls("moe_place", tokens, list(range(1, 17)), experts)
never_falls("embedding_grad", tokens, around(2, 512, 1 << 17, 1 << 18, (1 << 31) - 2), around(2, 8, 512, 1024, 1029, 7168, (1 << 24) - 1))
"""


@pytest.mark.parametrize("npes", [1, 2, 3, 8, 16, 64])
def test_workspaces_do_not_get_smaller(recorded, npes):  # noqa: F811
    """So that what a program allocates for its largest batch holds the smaller ones as well."""
    recorded(WORKSPACES % npes)


def test_a_workspace_of_the_largest_batch_serves_smaller_ones(recorded):  # noqa: F811
    """Workspaces that end where the PE's slice does: a call that needed more would be refused."""
    recorded("""
from nvshmem_amd import Runtime
rt = Runtime(npes=8, symmetric_size=1 << 30)
p = [rt.malloc(96 << 20) for _ in range(8)]
end = p[0] + rt.ptr(p[0], 1) - rt.ptr(p[0], 0) - 2048
launches()

def last(op, *sizes):
    return (end - rt.workspace_bytes(op, *sizes)) // 64 * 64

ws = last("moe_route", 8192, 256)
for t in (1, 64, 65, 1000, 1024, 2048, 2049, 5000, 8192):
    for e in (8, 64, 256):
        rt.moe_route("bfloat16", p[0], p[1], p[2], ws, p[3], t, e, 4, loss=p[4], balance=p[5])
ws = last("moe_route", 8192, 300)
for t in (1, 256, 512, 513, 1024, 4096, 8192):
    for e in (256, 257, 300):
        rt.moe_route("bfloat16", p[0], p[1], p[2], ws, p[3], t, e, 4, loss=p[4], balance=p[5])
ws = last("moe_place", 16384, 8, 256)
for t in (100, 1000, 8192, 16128, 16129, 16383, 16384):
    rt.moe_place(p[0], p[1], p[2], p[3], ws, p[4], p[5], t, 8, 256, 100)
ws = last("embedding_grad", 1207, 10003, 4096)
for t in (1, 100, 329, 600, 1206, 1207):
    for d in (1, 512, 1029, 4096):
        rt.embedding_grad("bfloat16", p[0], p[1], p[2], ws, t, 10003, d)
""")


def test_the_most_tokens_that_the_tables_take(recorded):  # noqa: F811
    """2^31 - 1 copies over all PEs; one token more is refused."""
    recorded("""
from nvshmem_amd import Runtime
from nvshmem_amd.host import NvshmemError
rt = Runtime(npes=4, symmetric_size=16 << 30)
tokens = (1 << 29) - 1
expert, dest_pe, dest_row = rt.malloc(tokens * 4), rt.malloc(tokens * 4), rt.malloc(tokens * 8)
counts, expected, expert_row = (rt.malloc(1025 * 8) for _ in range(3))
ws = rt.malloc(rt.workspace_bytes("moe_place", tokens, 1, 1024))
launches()
for experts in (4, 1024):
    rt.moe_place(dest_pe, dest_row, expected, expert_row, ws, expert, counts, tokens, 1, experts, 1 << 40)
    names = [l[0] for l in launches()]
    assert len(names) == 2 and "place_count" in names[0] and "place_kernel" in names[1], names
    try:
        rt.moe_place(dest_pe, dest_row, expected, expert_row, ws, expert, counts, tokens + 1, 1, experts, 1 << 40)
    except NvshmemError as e:
        assert "at most 2^31 - 1 in all" in str(e), str(e)
    else:
        raise AssertionError("not refused")
    assert not launches()
""")
