"""The experts' block where dim or hidden is at its most, on operands of which few elements are not zero, so that each one counts."""
import numpy as np
import pytest

import expert_bounds as B
from gpu_util import note, runtime
from token_util import Arrays, rounded

pytestmark = pytest.mark.gpu

MOST = 65536


def ends(k):
    """Where steps and tiles of a row begin and end, at its own ends and in its middle."""
    near = [1, 2, 64, 65, 128, 129, 256, 257]
    return np.array([0, 1, 31, 32, 63, 64, 127, 128, 255, 256, 32767, 32768] + [k - n for n in near])


def few(rng, rows, k):
    """Which elements are not zero: in every row of `k` three, at the ends of tiles and of the row among them; all of short rows."""
    if k < 1000:
        return np.ones((rows, k), bool)
    on = np.zeros((rows, k), bool)
    at, end = np.arange(rows), ends(k)
    on[at, end[at % len(end)]] = on[at, end[(at * 7 + 3) % len(end)]] = on[at, rng.integers(0, k, rows)] = True
    return on


@pytest.mark.parametrize("kind", ["bfloat16", "half", "float"])
@pytest.mark.parametrize("dim,hidden", [(MOST, 8), (8, MOST), (MOST - 1, 9), (9, MOST - 1)])
@pytest.mark.parametrize("rows", [35, 70])
def test_widest(kind, dim, hidden, rows):
    first, cap = 3, rows + 5
    rng = np.random.default_rng(dim + rows)
    table = np.array([[first, first + rows]])

    def numbers(shape, scale=1.0):
        return rounded(rng.standard_normal(shape) * scale, kind)

    x = np.where(few(rng, rows, dim), numbers((rows, dim)), 0).astype(np.float32)
    dout = np.where(few(rng, rows, dim), numbers((rows, dim)), 0).astype(np.float32)
    w_in, w_out = numbers((2 * hidden, dim)), numbers((dim, hidden), 0.3)
    on = few(rng, rows, hidden)
    pre = np.concatenate([np.where(on, numbers((rows, hidden)), 0), np.where(on, numbers((rows, hidden)), 0)], 1).astype(np.float32)
    if hidden > 1000:       # up is zero but for some columns, and so is h
        w_in[hidden + np.setdiff1d(np.arange(hidden), np.concatenate([ends(hidden), rng.integers(0, hidden, 30)]))] = 0

    def around(values):
        full = np.full((1, cap, values.shape[1]), np.nan, np.float32)
        full[0, first:first + rows] = values
        return full

    with runtime(1, 1 << 30) as rt, Arrays(rt) as new:
        er = new("int64", (2,), table)
        xa, da, pa = (new(kind, (cap, v.shape[1]), around(v)) for v in (x, dout, pre))
        wi, wo = new(kind, (1, 2 * hidden, dim), w_in[None, None]), new(kind, (1, dim, hidden), w_out[None, None])
        out, kept, drows = new(kind, (cap, dim)), new(kind, (cap, 2 * hidden)), new(kind, (cap, dim))
        dw_in, dw_out = new(kind, (1, 2 * hidden, dim)), new(kind, (1, dim, hidden))
        ws = new.workspace("moe_experts_grad", cap, 1, dim, hidden)
        note("widest", kind, dim, hidden, rows)
        rt.moe_experts(kind, out.address, ws.address, xa.address, wi.address, wo.address, er.address, cap, 1, dim, hidden, pre=kept.address)
        rt.moe_experts_grad(kind, drows.address, dw_in.address, dw_out.address, ws.address, da.address, xa.address, pa.address, wi.address,
                            wo.address, er.address, cap, 1, dim, hidden)
        rt.sync()
        ws.get()
        got = [a.get()[0] for a in (kept, out, drows, dw_in, dw_out)]
    own = slice(first, first + rows)
    results = B.forward(B.f64(x), B.f64(w_in), B.f64(w_out), kind) + B.backward(B.f64(dout), B.f64(x), B.f64(pre), B.f64(w_in), B.f64(w_out), kind)
    for name, g, (want, bound) in zip(("pre", "out", "drows", "dw_in", "dw_out"), got, results):
        B.close(g[0] if name.startswith("dw") else g[own], want, bound, name)
        # A zero in place of an element that is none is outside, but for small ones: sums of n of what is rounded by 2^-8 at most are bounded by
        # 0.64 n^0.5 2^-8 of their size, and as many elements and a fifth less are within that: 0.022 of them for the 50 columns of h here.
        passed = float((want.abs() <= bound)[want != 0].double().mean())
        assert passed < 0.03, name
