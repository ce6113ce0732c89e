"""The experts' block on the smallest numbers of its types, and on infinities and NaN."""
import numpy as np
import pytest

import expert_bounds as B
import expert_forms as F
from four_bit_util import ROWS, TABLE, call, values
from gpu_util import note, runtime
from token_util import Arrays, rounded

pytestmark = pytest.mark.gpu

# the smallest number is 2^LEAST and has so many bits above it before it is a normal one
LEAST = {"float": -149, "half": -24, "bfloat16": -133}
BITS = {"float": 23, "half": 10, "bfloat16": 7}


def subnormal(rng, kind, shape):
    v = rng.integers(1, 1 << BITS[kind], shape) * 2.0 ** LEAST[kind] * rng.choice([-1, 1], shape)
    assert np.array_equal(rounded(v, kind), v.astype(np.float32))
    return v.astype(np.float32)


def run(rt, new, kind, x, w_in, w_out, dout=None, pre=None):
    """out and pre, or drows, dw_in and dw_out, of experts that have ROWS."""
    cap, dim, hidden, mine = x.shape[0], x.shape[1], w_out.shape[2], len(ROWS)
    er, xa = new("int64", (mine + 1,), TABLE), new(kind, x.shape, x[None])
    wi, wo = new(kind, w_in.shape, w_in[None]), new(kind, w_out.shape, w_out[None])
    ws = new.workspace("moe_experts_grad", cap, mine, dim, hidden)
    note("extremes", kind, dim, hidden, dout is None)
    if dout is None:
        out, kept = new(kind, (cap, dim)), new(kind, (cap, 2 * hidden))
        rt.moe_experts(kind, out.address, ws.address, xa.address, wi.address, wo.address, er.address, cap, mine, dim, hidden, pre=kept.address)
        results = [out, kept]
    else:
        da, pa = new(kind, dout.shape, dout[None]), new(kind, pre.shape, pre[None])
        results = [new(kind, (cap, dim)), new(kind, w_in.shape), new(kind, w_out.shape)]
        rt.moe_experts_grad(kind, *[r.address for r in results], ws.address, da.address, xa.address, pa.address, wi.address, wo.address,
                            er.address, cap, mine, dim, hidden)
    rt.sync()
    ws.get()
    return [r.get()[0] for r in results]


@pytest.mark.parametrize("kind", F.KINDS)
@pytest.mark.parametrize("dim,hidden", [(136, 72), (135, 71)])
@pytest.mark.parametrize("small", ["rows", "weights"])
def test_smallest_numbers(kind, dim, hidden, small):
    """Elements below the least normal number, times what makes ordinary numbers of them."""
    rng = np.random.default_rng(dim)
    cap, mine = int(TABLE[0, -1]), len(ROWS)
    up = 2.0 ** (-LEAST[kind] - BITS[kind])         # 2^126; 2^14

    def ordinary(shape, scale=1.0):
        return rounded(rng.standard_normal(shape) * scale, kind)

    def large(shape):
        return rounded(rng.uniform(0.5, 1, shape) * rng.choice([-1, 1], shape) * up, kind)

    x, w_in = (subnormal, large)[small == "weights"], (subnormal, large)[small == "rows"]
    x, w_in = (f(*((rng, kind) if f is subnormal else ()), s) for f, s in ((x, (cap, dim)), (w_in, (mine, 2 * hidden, dim))))
    w_out = ordinary((mine, dim, hidden), hidden ** -0.5)
    with runtime(1, 64 << 20) as rt, Arrays(rt) as new:
        out, kept = run(rt, new, kind, x, w_in, w_out)
        # the way back: dout or the second product's weights
        dout, w_back = (subnormal(rng, kind, (cap, dim)), large((mine, dim, hidden))) if small == "rows" else (
            large((cap, dim)), subnormal(rng, kind, (mine, dim, hidden)))
        pre = ordinary((cap, 2 * hidden), 1.5)
        w_first, rows = ordinary((mine, 2 * hidden, dim), 0.1), ordinary((cap, dim), 0.1)
        drows, dw_in, dw_out = run(rt, new, kind, rows, w_first, w_back, dout, pre)
    for i in range(mine):
        own = slice(*TABLE[0, i:i + 2])
        what = " of %d rows" % ROWS[i]
        (want_pre, pre_bound), (want, bound) = B.forward(B.f64(x[own]), B.f64(w_in[i]), B.f64(w_out[i]), kind)
        B.close(kept[own], want_pre, pre_bound, "pre" + what)
        B.close(out[own], want, bound, "out" + what)
        (want, bound), (want_in, bound_in), (want_out, bound_out) = B.backward(B.f64(dout[own]), B.f64(rows[own]), B.f64(pre[own]),
                                                                               B.f64(w_first[i]), B.f64(w_back[i]), kind)
        B.close(drows[own], want, bound, "drows" + what)
        B.close(dw_in[i], want_in, bound_in, "dw_in" + what)
        if small == "rows":     # (else beyond the largest number of a half)
            # sums of subnormal numbers of fp32: every product and every addition is off by up to 2^-149
            slack = 2 * (own.stop - own.start) * 2.0 ** -149 if kind != "half" else 0
            B.close(dw_out[i], want_out, bound_out + slack, "dw_out" + what)


@pytest.mark.parametrize("kind", F.KINDS)
@pytest.mark.parametrize("dim,hidden", [(136, 72), (135, 71)])
def test_infinities_and_nans(kind, dim, hidden):
    """They come out where the formula has them, and nowhere else."""
    rng = np.random.default_rng(hidden)
    cap, mine = int(TABLE[0, -1]), len(ROWS)

    def numbers(shape, scale=1.0):
        return rounded(rng.standard_normal(shape) * scale, kind)

    plain = numbers((cap, dim))
    special = np.arange(cap) % 7 == 0
    x = plain.copy()
    for n, row in enumerate(np.flatnonzero(special)):
        x[row, rng.integers(dim)] = [np.inf, -np.inf, np.nan][n % 3]
    w_in, w_out = numbers((mine, 2 * hidden, dim), dim ** -0.5), numbers((mine, dim, hidden), hidden ** -0.5)
    w_in[:, :hidden] = np.abs(w_in[:, :hidden])     # gate goes to the infinity that a row has
    w_out[:, ::2] = 0
    w_out[:, ::2, hidden // 2] = 1                  # one element of h, and zeros times the others
    dout, pre = numbers((cap, dim)), numbers((cap, 2 * hidden))
    bad_dout = dout.copy()
    bad_dout[special, rng.integers(0, dim, special.sum())] = np.inf
    with runtime(1, 64 << 20) as rt, Arrays(rt) as new:
        out, kept = run(rt, new, kind, x, w_in, w_out)
        again, kept_again = run(rt, new, kind, plain, w_in, w_out)
        drows = run(rt, new, kind, plain, w_in, w_out, bad_dout, pre)[0]
        drows_again = run(rt, new, kind, plain, w_in, w_out, dout, pre)[0]
    for got, other in ((out, again), (kept, kept_again), (drows, drows_again)):
        assert np.array_equal(got[~special], other[~special])
    for i in range(mine):
        own = np.arange(*TABLE[0, i:i + 2])
        own = own[special[own]]
        if len(own) == 0:
            continue
        (want_pre, pre_bound), (want, bound) = B.forward(B.f64(x[own]), B.f64(w_in[i]), B.f64(w_out[i]), kind)
        B.close(kept[own], want_pre, pre_bound.nan_to_num(), "pre")
        B.close(out[own], want, bound.nan_to_num(), "out")
        want, bound = B.backward(B.f64(bad_dout[own]), B.f64(plain[own]), B.f64(pre[own]), B.f64(w_in[i]), B.f64(w_out[i]), kind)[0]
        B.close(drows[own], want, bound.nan_to_num(), "drows")


@pytest.mark.parametrize("kind", F.KINDS)
@pytest.mark.parametrize("group", [32, 128])
def test_small_rows_times_four_bits(kind, group):
    """Rows of the smallest numbers of 16-bit types; of fp32 ones whose last bits are above 2^-133."""
    mine, dim, hidden, cap = len(ROWS), 264, 72, int(TABLE[0, -1])
    rng = np.random.default_rng(group)
    if kind == "float":
        x, up = rounded(rng.standard_normal((1, cap, dim)) * 2.0 ** -100, kind), 2.0 ** 100
        x[np.abs(x) < 2.0 ** -109] = 0
    else:
        x, up = subnormal(rng, kind, (1, cap, dim)), 2.0 ** (-LEAST[kind] - BITS[kind])
    q_in, q_out = rng.integers(0, 16, (1, mine, 2 * hidden, dim)), rng.integers(0, 16, (1, mine, dim, hidden))
    s_in = rounded(rng.uniform(0.5, 1, (1, mine, 2 * hidden, -(-dim // group))) * up / 16, kind)
    s_out = rounded(rng.uniform(0.01, 0.03, (1, mine, dim, -(-hidden // group))), kind)
    with runtime(1, 64 << 20) as rt, Arrays(rt) as new:
        got = call(rt, new, kind, x, q_in, s_in, q_out, s_out, TABLE, group)

    def scales(s, k):
        return B.f64(s.astype(np.float64)[:, np.arange(k) // group])

    for i in range(mine):
        own = slice(*TABLE[0, i:i + 2])
        want, bound = B.forward_four_bits(B.f64(x[0, own]), B.f64(values(q_in[0, i], s_in[0, i], group)), scales(s_in[0, i], dim),
                                          B.f64(values(q_out[0, i], s_out[0, i], group)), scales(s_out[0, i], hidden), kind, group)
        assert want.abs().max() > 0.1
        B.close(got[0, own], want, bound, "expert of %d rows" % ROWS[i])
