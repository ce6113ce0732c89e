"""The experts' block with weights of 4 bits on rows that are large, infinite, or of one sign."""
import numpy as np
import pytest

import expert_reference as R
from four_bit_util import ROWS, TABLE, call, values
from gpu_util import runtime
from token_util import Arrays, close, rounded

pytestmark = pytest.mark.gpu


def expected(x, w_in, w_out, kind):
    _, _, want, bound = R.forward(R.f64(x), R.f64(w_in), R.f64(w_out), kind)
    return want.numpy(), bound.numpy()


@pytest.mark.parametrize("kind", ["bfloat16", "float"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("power", [114, 117, 120])
def test_large_elements_of_one_sign(kind, group, power):
    """Rows that are ordinary in the first half of dim, and rows that are large in the second, whose scales are as small: results of the
    same size, whatever the number of rows that came with them.  Sums of 128 products of q - 8 and elements under 2^121 leave fp32,
    sixteenths of them stay under 2^127."""
    mine, dim, hidden, cap = len(ROWS), 256, 72, int(TABLE[0, -1])
    rng = np.random.default_rng(group + power)
    large = np.arange(cap) % 3 == 0
    x = np.zeros((1, cap, dim), np.float32)
    x[0, ~large, :128] = rng.standard_normal(((~large).sum(), 128))
    x[0, large, 128:] = rng.uniform(1, 1.99, (large.sum(), 128)) * 2.0 ** power
    x = rounded(x, kind)
    q_in, q_out = rng.integers(0, 16, (1, mine, 2 * hidden, dim)), rng.integers(0, 16, (1, mine, dim, hidden))
    q_in[0, :, 5], q_in[0, :, hidden + 5] = 0, 0       # (the largest sum that there is)
    s_in = rng.uniform(0.01, 0.03, (1, mine, 2 * hidden, dim // group))
    s_in[..., 128 // group:] *= 2.0 ** -power
    s_in, s_out = rounded(s_in, kind), rounded(rng.uniform(0.01, 0.03, (1, mine, dim, -(-hidden // group))), kind)
    with runtime(1, 64 << 20) as rt, Arrays(rt) as new:
        got = call(rt, new, kind, x, q_in, s_in, q_out, s_out, TABLE, group)
        # without the large rows, every other row's bits
        other = np.where(large[None, :, None], np.float32(0), x)
        again = call(rt, new, kind, other, q_in, s_in, q_out, s_out, TABLE, group)
    assert np.array_equal(got[0, ~large], again[0, ~large])
    for i in range(mine):
        rows = np.arange(TABLE[0, i], TABLE[0, i + 1])
        rows = rows[large[rows]]
        if len(rows):
            want, bound = expected(x[0, rows], values(q_in[0, i], s_in[0, i], group), values(q_out[0, i], s_out[0, i], group), kind)
            assert np.isfinite(want).all()
            close(got[0, rows], want, bound, "expert of %d rows" % ROWS[i])


@pytest.mark.parametrize("kind", ["bfloat16", "half", "float"])
@pytest.mark.parametrize("group", [32, 128])
def test_infinite_elements(kind, group):
    """An infinity goes through the products as the definition says: times weights of one sign it is one, times a weight of 0, or added to
    its negative, a NaN.  The other rows do not know of it."""
    mine, dim, hidden, cap = len(ROWS), 264, 40, int(TABLE[0, -1])
    rng = np.random.default_rng(group)
    ordinary = rounded(rng.standard_normal((1, cap, dim)), kind)
    special = np.arange(cap) % 5 == 0
    x = ordinary.copy()
    for n, row in enumerate(np.flatnonzero(special)):
        x[0, row, rng.integers(dim)] = [np.inf, np.inf, np.nan, -np.inf][n % 4]
    q_in = rng.integers(9, 16, (1, mine, 2 * hidden, dim))      # gate: positive everywhere
    sign = rng.integers(0, 2, (1, mine, hidden))                # up: of one sign in a row
    q_in[:, :, hidden:] = np.where(sign[..., None], q_in[:, :, hidden:], q_in[:, :, hidden:] - 9)
    q_out = rng.integers(9, 16, (1, mine, dim, hidden))         # out: of up's signs in every second row, which adds up to an infinity
    q_out = np.where(sign[:, :, None], q_out, q_out - 9)
    q_out[:, :, 1::2] = rng.integers(0, 16, q_out[:, :, 1::2].shape)
    s_in = rounded(rng.uniform(0.01, 0.02, (1, mine, 2 * hidden, -(-dim // group))), kind)
    s_out = rounded(rng.uniform(0.01, 0.02, (1, mine, dim, -(-hidden // group))), kind)
    with runtime(1, 64 << 20) as rt, Arrays(rt) as new:
        got = call(rt, new, kind, x, q_in, s_in, q_out, s_out, TABLE, group)
        again = call(rt, new, kind, ordinary, q_in, s_in, q_out, s_out, TABLE, group)
    assert np.array_equal(got[0, ~special], again[0, ~special])
    infinite = 0
    for i in range(mine):
        rows = np.arange(TABLE[0, i], TABLE[0, i + 1])
        rows = rows[special[rows]]
        if len(rows):
            want, bound = expected(x[0, rows], values(q_in[0, i], s_in[0, i], group), values(q_out[0, i], s_out[0, i], group), kind)
            infinite += np.isinf(want).sum()
            close(got[0, rows], want, np.nan_to_num(bound), "expert of %d rows" % ROWS[i])
    assert infinite
