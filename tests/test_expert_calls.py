"""What the experts' block and dropout refuse, and that a refused call enqueues nothing: seen on the CPU, where nothing runs."""
import pytest

from launch_recorder import recorded  # noqa: F401
from test_token_calls import SETUP

EXPERTS = SETUP + """
E, D, H, CAP = 8, 24, 16, 30
def at(i, value, call, base, **more):
    args = list(base)
    args[i] = value
    refused(call, *args, **more)

def check(call, base, names, written, aligned):
    for i, name in enumerate(names, 1):
        at(i, None, call, base, text="%s %s" % (call.__name__, name))
        at(i, 0x1234, call, base, text="not a symmetric address")
        at(i, END - 16, call, base, text="leave")
        if aligned.get(name, 4) > 1:
            at(i, base[i] + aligned.get(name, 4) // 2, call, base, text="aligned")
        if name in written:
            for j in range(1, len(names) + 1):
                if j != i:
                    at(i, base[j], call, base, text="overlaps")
    first = len(names) + 1      # recv_cap_rows, experts, dim, hidden
    for cap in (1 << 40, 1 << 63):
        at(first, cap, call, base, text="leave")
    for experts in (0, -4, 1028):
        at(first + 1, experts, call, base, text="experts")
    at(first + 1, 6, call, base, text="same number")
    for size in (0, 65537, 1 << 40):
        at(first + 2, size, call, base, text="elements")
        at(first + 3, size, call, base, text="elements")

names = ("out", "workspace", "rows", "w_in", "w_out", "expert_row")
good = ("float", A[0], A[1], A[2], A[3], A[4], A[5], CAP, E, D, H)
assert len(taken(rt.moe_experts, *good)) == 2
check(rt.moe_experts, good, names, ("out", "workspace"), {"workspace": 64, "expert_row": 8})
assert len(taken(rt.moe_experts, *good, pre=A[6])) == 2
refused(rt.moe_experts, *good, pre=A[0], text="overlaps")
refused(rt.moe_experts, *good, pre=A[2], text="overlaps")
refused(rt.moe_experts, *good, pre=0x1234, text="not a symmetric address")
assert taken(rt.moe_experts, "half", None, None, None, A[3], A[4], A[5], 0, E, D, H) == []
assert len(taken(rt.moe_experts, "half", A[0] + 2, A[1], A[2] + 6, A[3] + 2, A[4] + 2, A[5], CAP, E, D, H)) == 2

names = ("drows", "dw_in", "dw_out", "workspace", "dout", "rows", "pre", "w_in", "w_out", "expert_row")
good = ("bfloat16",) + tuple(A[:10]) + (CAP, E, D, H)
assert len(taken(rt.moe_experts_grad, *good)) == 4
check(rt.moe_experts_grad, good, names, ("drows", "dw_in", "dw_out", "workspace"), dict({n: 2 for n in names}, workspace=64, expert_row=8))
# without rows there is nothing but zeros to write
assert len(taken(rt.moe_experts_grad, "float", None, A[1], A[2], None, None, None, None, A[7], A[8], A[9], 0, E, D, H)) == 2

names = ("out", "workspace", "rows", "w_in", "w_in_scale", "w_out", "w_out_scale", "expert_row")
good = ("float",) + tuple(A[:8]) + (CAP, E, D, H, 32)
assert len(taken(rt.moe_experts_w4, *good)) == 2        # at most 64 rows an expert: no tiles
assert len(taken(rt.moe_experts_w4, "float", *A[:8], 100, E, D, H, 64)) == 4
check(rt.moe_experts_w4, good, names, ("out", "workspace"), {"workspace": 64, "expert_row": 8, "w_in": 1, "w_out": 1})
for group in (0, -32, 16, 48, 33, 65536 + 32, 1 << 30):
    refused(rt.moe_experts_w4, *good[:-1], group, text="groups")
assert taken(rt.moe_experts_w4, "half", None, None, None, *A[3:8], 0, E, D, H, 128) == []
"""

DROPOUT = SETUP + """
T, D = 10, 40
good = ("float", A[0], A[1], A[2], T, D, 0.1)
assert len(taken(rt.dropout, *good)) == 1
def at(i, value, **more):
    args = list(good)
    args[i] = value
    refused(rt.dropout, *args, **more)
for i, name in ((1, "out"), (2, "rows"), (3, "seed")):
    at(i, None, text="dropout %s" % name)
    at(i, 0x1234, text="not a symmetric address")
    at(i, A[i - 1] + 2, text="aligned")
at(1, END - 64, text="leave")
at(1, A[2], text="overlaps")
at(1, A[1] + 4, text="overlaps")
assert len(taken(rt.dropout, "float", A[1], A[1], A[2], T, D, 0.1)) == 1                        # in place
refused(rt.dropout, *good, residual=0x1234, text="not a symmetric address")
refused(rt.dropout, "float", A[1], A[1], A[2], T, D, 0.1, residual=A[3], text="overlaps rows")
assert len(taken(rt.dropout, "float", A[3], A[1], A[2], T, D, 0.1, residual=A[3])) == 1         # onto the residual
for p in (-0.1, 1.0, 1.5, 0.999999, float("nan"), float("inf")):
    at(6, p, text="probability")
at(4, 1 << 40, text="leave")
at(4, 1 << 63, text="leave")
at(5, 0, text="elements")
at(5, (1 << 24) + 1, text="elements")
assert taken(rt.dropout, "half", None, None, A[2], 0, D, 0.5) == []
"""


@pytest.mark.parametrize("code", [EXPERTS, DROPOUT], ids=["experts", "dropout"])
def test_refusals(recorded, code):  # noqa: F811
    recorded(code)


def test_before_init(recorded):  # noqa: F811
    recorded("""
for t in ("float", "half", "bfloat16"):
    assert getattr(lib, "nvshmemx_amd_%s_moe_experts_on_stream" % t)(1, 1, 1, 1, 1, 1, 1, 1, 8, 1, 1, None) != 0
    assert b"before nvshmem_init" in lib.nvshmemx_amd_last_error()
    assert getattr(lib, "nvshmemx_amd_%s_dropout_on_stream" % t)(1, 1, 1, 1, 1, 1, 0.5, None) != 0
assert lib.nvshmemx_amd_moe_experts_workspace(10, 8, 10, 10) == 0
assert lib.nvshmemx_amd_moe_experts_grad_workspace(10, 8, 10, 10) == 0
assert not launches()
""")


def test_no_grid_leaves_its_limits(recorded):  # noqa: F811
    """A launch holds fewer than 2^32 threads, in at most 65535 blocks along y and z (the recorder refuses others)."""
    recorded("""
from nvshmem_amd import Runtime
rt = Runtime(npes=4, symmetric_size=100 << 30)
p = [rt.malloc(4 << 30) for _ in range(20)]
launches()
for dim, hidden, experts, cap in ((65536, 1, 1024, 30000), (1, 65536, 1024, 2000), (1, 1, 1024, (1 << 30) - 1), (1, 1, 4, (1 << 30) - 1),
                                  (65536, 65536, 4, 70), (4096, 4096, 4, 200000)):
    big = [a for a in p[::4]]
    for t in ("half",):
        try:
            rt.moe_experts(t, p[0], p[1], p[2], p[3], p[7], p[11], cap, experts, dim, hidden)
            rt.moe_experts_w4(t, p[0], p[1], p[2], p[3], p[7], p[8], p[12], p[13], cap, experts, dim, hidden, 32)
        except Exception as e:
            assert "overlaps" in str(e) or "leave" in str(e), str(e)
assert launches()
rt.dropout("half", p[0], p[2], p[4], (1 << 31) - 64, 1, 0.5)
rt.dropout("half", p[0], p[2], p[4], 100, 1 << 24, 0.5)
rt = None
""")
    recorded("""
from nvshmem_amd import Runtime
rt = Runtime(npes=64, symmetric_size=4 << 30)
a, b, s = rt.malloc(1 << 30), rt.malloc(1 << 30), rt.malloc(16)
launches()
rt.dropout("half", a, b, s, 1 << 29, 1, 0.5)
assert len(launches()) == 1
""")


@pytest.mark.parametrize("npes", [1, 8])
def test_workspaces_do_not_get_smaller(recorded, npes):  # noqa: F811
    """... and serve every type, in both forms."""
    recorded("""
import itertools
from nvshmem_amd import Runtime
rt = Runtime(npes=%d, symmetric_size=1 << 30)
grids = [[0, 1, 7, 64, 1000, 1 << 20], [8, 64, 1024], [1, 64, 7168, 65536], [1, 33, 2048, 65536]]
for op in ("moe_experts", "moe_experts_grad"):
    size = {p: rt.workspace_bytes(op, *p) for p in itertools.product(*grids)}
    for p, n in size.items():
        for i, grid in enumerate(grids):
            q = p[:i] + (grid[max(grid.index(p[i]) - 1, 0)],) + p[i + 1:]
            assert size[q] <= n
# a workspace at the end of what may be used, for smaller batches
room = rt.malloc(200 << 20)
p = [room + i * (10 << 20) for i in range(18)]
end = room + (rt.ptr(room, 1) - rt.ptr(room, 0) if rt.npes > 1 else (1 << 30) + 2048 + (16 << 20) - ((1 << 30) + 2048) %% (16 << 20)) - 2048
for op in ("moe_experts", "moe_experts_grad"):
    ws = (end - rt.workspace_bytes(op, 300, 8, 64, 333)) // 64 * 64
    for kind in ("float", "half"):
        for cap in (1, 100, 299, 300):
            for hidden in (1, 64, 333):
                if op == "moe_experts":
                    rt.moe_experts(kind, p[0], ws, p[1], p[2], p[3], p[4], cap, 8, 64, hidden)
                    rt.moe_experts_w4(kind, p[0], ws, p[1], p[2], p[3], p[4], p[5], p[6], cap, 8, 64, hidden, 32)
                else:
                    rt.moe_experts_grad(kind, p[0], p[1], p[2], ws, *p[3:9], cap, 8, 64, hidden)
""" % npes)


def test_shapes_of_tiles(recorded):  # noqa: F811
    """Which tiles the sizes lead to: (rows, columns) in the kernels' names."""
    recorded(SETUP.replace("8 << 20", "512 << 20") + """
import re
def shapes(call, *args):
    call(*args)
    return [tuple(int(v) for v in re.search(r"Lj(\\d+)ELj(\\d+)E", l[0]).groups()) for l in launches()]

room = rt.malloc(400 << 20)
p = [room + i * (38 << 20) for i in range(10)]
large = dict(mine=16, cap=16 * 460, dim=776, hidden=776)        # as in test_gpu_experts.py, there on two PEs
E = 32                                                          # (of all PEs: eight on each of the four here)
for kind, want in (("bfloat16", (256, 256)), ("half", (256, 256)), ("float", (64, 128))):
    assert shapes(rt.moe_experts, kind, *p[:6], 8 * 460, E, large["dim"], large["hidden"]) == [want] * 2, kind
    got = shapes(rt.moe_experts_grad, kind, *p[:10], 8 * 460, E, large["dim"], large["hidden"])
    assert got == [want] * 2 + [want if kind != "float" else (128, 128)] * 2, (kind, got)
# rows of an expert, with tiles enough for the GPU: 64 experts of 1024 x 1024
for cap, want in ((16 * 12, (32, 128)), (16 * 13, (64, 128)), (16 * 32, (64, 128)), (16 * 33, (128, 128)), (16 * 448, (128, 128)), (16 * 449, (256, 256))):
    assert shapes(rt.moe_experts, "half", *p[:6], cap, 64, 512, 1024)[0] == want, cap
# ... and without
assert shapes(rt.moe_experts, "half", *p[:6], 40, 4, 512, 256) == [(32, 128)] * 2
assert shapes(rt.moe_experts, "half", *p[:6], 900, 4, 512, 256) == [(32, 128)] * 2
assert shapes(rt.moe_experts, "half", *p[:6], 1000, 4, 512, 256) == [(64, 128)] * 2
# rows that no vector divides have no tiles of 256 rows
assert shapes(rt.moe_experts, "half", *p[:6], 16 * 460, 64, 511, 1024)[0] == (128, 128)
""")
