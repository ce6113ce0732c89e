"""The experts' gated feed-forward block and its gradients against 64 bits."""
import numpy as np
import pytest
import torch

import expert_reference as R
from gpu_util import note, runtime
from token_util import Arrays, close, rounded

pytestmark = pytest.mark.gpu

KINDS = ["bfloat16", "half", "float"]


def starts(npes, mine, cap, sizes, rng, first=0):
    """expert_row of every PE: the experts have rows of `sizes` in an order of their own, as far as there is room."""
    rows = np.zeros((npes, mine + 1), np.int64)
    for pe in range(npes):
        n = rng.permutation(np.resize(sizes, mine))
        rows[pe] = np.minimum(first + np.concatenate([[0], np.cumsum(n)]), cap)
    return rows


class Case:
    """Operands of a call; rows that no expert has are NaN."""

    def __init__(self, new, rng, kind, npes, mine, cap, dim, hidden, expert_row, shift=0):
        self.kind, self.npes, self.mine, self.cap, self.dim, self.hidden = kind, npes, mine, cap, dim, hidden
        self.expert_row = expert_row
        self.er = new("int64", (mine + 1,), expert_row)
        busy = np.zeros((npes, cap, 1), bool)
        for pe in range(npes):
            for a, b in R.ranges(expert_row[pe], cap):
                busy[pe, a:b] = True
        self.busy = busy[..., 0]

        def rows(width, scale=1.0):
            v = np.where(busy, rounded(rng.standard_normal((npes, cap, width)) * scale, kind), np.nan).astype(np.float32)
            return v, new(kind, (cap, width), v, shift)

        self.rows = rows
        self.w_in_values = rounded(rng.standard_normal((npes, mine, 2 * hidden, dim)) / np.sqrt(dim), kind)
        self.w_out_values = rounded(rng.standard_normal((npes, mine, dim, hidden)) / np.sqrt(hidden), kind)
        self.w_in = new(kind, (mine, 2 * hidden, dim), self.w_in_values, shift)
        self.w_out = new(kind, (mine, dim, hidden), self.w_out_values, shift)
        self.x_values, self.x = rows(dim)

    def each(self):
        for pe in range(self.npes):
            for i, (a, b) in enumerate(R.ranges(self.expert_row[pe], self.cap)):
                yield pe, i, a, b


def check_forward(rt, new, c, with_pre, shift=0):
    out = new(c.kind, (c.cap, c.dim), None, shift)
    pre = new(c.kind, (c.cap, 2 * c.hidden), None, shift) if with_pre else None
    ws = new.workspace("moe_experts", c.cap, c.mine * c.npes, c.dim, c.hidden)
    untouched = out.get()
    note("moe_experts", c.kind, c.npes, c.mine, c.cap, c.dim, c.hidden, c.expert_row.tolist())
    rt.moe_experts(c.kind, out.address, ws.address, c.x.address, c.w_in.address, c.w_out.address, c.er.address, c.cap,
                   c.mine * c.npes, c.dim, c.hidden, pre=pre.address if pre else None)
    rt.sync()
    ws.get()
    got, got_pre = out.get(), pre.get() if pre else None
    for pe, i, a, b in c.each():
        want_pre, pre_bound, want, bound = R.forward(R.f64(c.x_values[pe, a:b]), R.f64(c.w_in_values[pe, i]),
                                                     R.f64(c.w_out_values[pe, i]), c.kind)
        close(got[pe, a:b], want, bound, "out of expert %d of PE %d" % (i, pe))
        if pre:
            close(got_pre[pe, a:b], want_pre, pre_bound, "pre of expert %d of PE %d" % (i, pe))
    assert np.array_equal(got[~c.busy], untouched[~c.busy])
    if pre:
        assert np.array_equal(got_pre[~c.busy].view(np.uint32), np.resize(untouched.reshape(-1)[:1], got_pre[~c.busy].shape).view(np.uint32))
    return got


def check_backward(rt, new, c, shift=0):
    dout_values, dout = c.rows(c.dim, 0.5)
    pre_values, pre = c.rows(2 * c.hidden, 1.5)
    drows = new(c.kind, (c.cap, c.dim), None, shift)
    dw_in, dw_out = new(c.kind, (c.mine, 2 * c.hidden, c.dim), None, shift), new(c.kind, (c.mine, c.dim, c.hidden), None, shift)
    ws = new.workspace("moe_experts_grad", c.cap, c.mine * c.npes, c.dim, c.hidden)
    untouched = drows.get()
    note("moe_experts_grad", c.kind, c.npes, c.mine, c.cap, c.dim, c.hidden, c.expert_row.tolist())
    rt.moe_experts_grad(c.kind, drows.address, dw_in.address, dw_out.address, ws.address, dout.address, c.x.address, pre.address,
                        c.w_in.address, c.w_out.address, c.er.address, c.cap, c.mine * c.npes, c.dim, c.hidden)
    rt.sync()
    ws.get()
    got, got_in, got_out = drows.get(), dw_in.get(), dw_out.get()
    for pe, i, a, b in c.each():
        (want, bound), (want_in, bound_in), (want_out, bound_out) = R.backward(
            R.f64(dout_values[pe, a:b]), R.f64(c.x_values[pe, a:b]), R.f64(pre_values[pe, a:b]), R.f64(c.w_in_values[pe, i]),
            R.f64(c.w_out_values[pe, i]), c.kind)
        what = " of expert %d of PE %d" % (i, pe)
        close(got[pe, a:b], want, bound, "drows" + what)
        close(got_in[pe, i], want_in, bound_in, "dw_in" + what)
        close(got_out[pe, i], want_out, bound_out, "dw_out" + what)
        if a == b:
            assert not got_in[pe, i].any() and not got_out[pe, i].any()
    assert np.array_equal(got[~c.busy], untouched[~c.busy])


SIZES = [(64, 64), (1, 1), (8, 16), (7, 3), (40, 24), (129, 70), (264, 136), (515, 129), (512, 384), (72, 1032)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,hidden", SIZES)
def test_sizes(kind, dim, hidden):
    npes, mine, cap = 2, 5, 411
    rng = np.random.default_rng(dim * 1000 + hidden)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        c = Case(new, rng, kind, npes, mine, cap, dim, hidden, starts(npes, mine, cap, [0, 1, 37, 300, 17], rng, 3))
        check_forward(rt, new, c, True)
        check_forward(rt, new, c, False)
        check_backward(rt, new, c)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes", [[0], [1], [15, 16], [17, 32, 33], [63, 65], [127, 128, 129], [255, 256, 257], [600, 0, 0, 1]])
def test_rows_of_an_expert(kind, sizes):
    npes, mine, dim, hidden = 3, 4, 136, 200
    rng = np.random.default_rng(sum(sizes) + 1)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        cap = sum(int(v) for v in np.resize(sizes, mine)) + 9
        c = Case(new, rng, kind, npes, mine, cap, dim, hidden, starts(npes, mine, cap, sizes, rng))
        check_forward(rt, new, c, True)
        check_backward(rt, new, c)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shift", [1, 3])
def test_operands_on_any_element(kind, shift):
    npes, mine, cap, dim, hidden = 2, 3, 150, 264, 72
    rng = np.random.default_rng(shift)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        c = Case(new, rng, kind, npes, mine, cap, dim, hidden, starts(npes, mine, cap, [70, 5, 40], rng, 2), shift)
        check_forward(rt, new, c, True, shift)
        check_backward(rt, new, c, shift)


@pytest.mark.parametrize("npes,mine", [(1, 1), (1, 130), (5, 2), (16, 1), (64, 1)])
def test_numbers_of_pes_and_experts(npes, mine):
    cap, dim, hidden = 200, 48, 40
    rng = np.random.default_rng(npes)
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        c = Case(new, rng, "bfloat16", npes, mine, cap, dim, hidden, starts(npes, mine, cap, [0, 3, 0, 1, 20, 0, 0, 2], rng))
        check_forward(rt, new, c, True)
        check_backward(rt, new, c)


def test_tables_that_leave_the_buffer():
    npes, cap, dim, hidden = 2, 90, 64, 64
    rng = np.random.default_rng(5)
    rows = np.array([[-7, 20, 20, 2 ** 40, 2 ** 62], [-2 ** 62, -5, 30, 90, -1]], np.int64)
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        c = Case(new, rng, "bfloat16", npes, 4, cap, dim, hidden, rows)
        check_forward(rt, new, c, True)
        check_backward(rt, new, c)


def test_no_rows_at_all():
    npes, mine, dim, hidden = 2, 3, 24, 40
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        c = Case(new, np.random.default_rng(0), "half", npes, mine, 0, dim, hidden, np.zeros((npes, mine + 1), np.int64))
        dw_in, dw_out = new("half", (mine, 2 * hidden, dim)), new("half", (mine, dim, hidden))
        note("no rows")
        rt.moe_experts("half", None, None, None, c.w_in.address, c.w_out.address, c.er.address, 0, mine * npes, dim, hidden)
        rt.moe_experts_grad("half", None, dw_in.address, dw_out.address, None, None, None, None, c.w_in.address, c.w_out.address,
                            c.er.address, 0, mine * npes, dim, hidden)
        rt.sync()
        assert not dw_in.get().any() and not dw_out.get().any()


def test_equal_inputs_give_equal_bits():
    npes, mine, cap, dim, hidden = 4, 4, 700, 320, 264
    rng = np.random.default_rng(9)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        c = Case(new, rng, "half", npes, mine, cap, dim, hidden, starts(npes, mine, cap, [300, 9, 150, 0], rng))
        first = check_forward(rt, new, c, False)
        for _ in range(3):
            assert np.array_equal(check_forward(rt, new, c, False), first, equal_nan=True)


# Experts of so many rows that every product takes the largest tiles (test_expert_calls.py holds them to that).
LARGE = dict(npes=2, mine=16, cap=16 * 460, dim=776, hidden=776)


@pytest.mark.parametrize("kind", ["bfloat16", "half"])
def test_largest_tiles(kind):
    rng = np.random.default_rng(12)
    with runtime(LARGE["npes"], 512 << 20) as rt, Arrays(rt) as new:
        sizes = [1000, 700, 3, 0, 257, 500, 512, 700, 460, 461, 600, 300, 256, 900, 127, 553]
        c = Case(new, rng, kind, expert_row=starts(LARGE["npes"], LARGE["mine"], LARGE["cap"], sizes, rng, 5), **LARGE)
        check_forward(rt, new, c, True)
        check_backward(rt, new, c)
