"""The experts' block with weights of 4 bits where much that is large adds up to little."""
import numpy as np
import pytest

import expert_reference as R
from four_bit_util import ROWS, TABLE, call, values
from gpu_util import runtime
from token_util import EPS, TINY, Arrays, close, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bfloat16", "half", "float"])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
def test_rows_of_one_sign_that_cancel(kind, group):
    """Whole numbers of one sign and of as many bits as the type has, in equal pairs, times weights that are opposite in all pairs but one.
    Every partial sum of q - 8 and elements is a whole number of less than 24 bits and so exact in fp32 (float: 16 bits of element)."""
    mine, dim, hidden, cap = len(ROWS), 512, 64, int(TABLE[0, -1])
    bits = {"bfloat16": 8, "half": 11, "float": 12}[kind]
    rng = np.random.default_rng(group)
    x = np.repeat(rng.integers(2 ** (bits - 1), 2 ** bits, (1, cap, dim // 2)), 2, -1).astype(np.float32)
    assert np.array_equal(x, rounded(x, kind))
    q_in = np.full((1, mine, 2 * hidden, dim), 8)
    q_in[:, :, :hidden, 0] = 9                                  # gate: the first element
    up = rng.integers(1, 8, (1, mine, hidden, dim // 2))
    q_in[:, :, hidden:, 0::2], q_in[:, :, hidden:, 1::2] = 8 + up, 8 - up
    column = rng.integers(0, dim // 2, hidden)                  # up: one element, once
    q_in[:, :, hidden + np.arange(hidden), 2 * column + 1] += 1
    q_out = np.full((1, mine, dim, hidden), 8)
    q_out[:, :, np.arange(dim), np.arange(dim) % hidden] = 9    # out: h
    # (powers of two, so that products with them are exact)
    s_in, s_out = np.full((1, mine, 2 * hidden, dim // group), 2.0 ** -bits), np.full((1, mine, dim, -(-hidden // group)), 1.0)
    with runtime(1, 64 << 20) as rt, Arrays(rt) as new:
        got = call(rt, new, kind, x, q_in, s_in, q_out, s_out, TABLE, group)
    for i in range(mine):
        rows = x[0, TABLE[0, i]:TABLE[0, i + 1]].astype(np.float64)
        w_in = values(q_in[0, i], s_in[0, i], group)
        gate, up = (rows @ w_in.T)[:, :hidden], (rows @ w_in.T)[:, hidden:]
        assert np.array_equal(up, rows[:, 2 * column] * 2.0 ** -bits)
        h = gate / (1 + np.exp(-gate)) * up
        # h: 16 half steps of fp32 for sigmoid and what is multiplied, and its rounding.  out: one element of h, in bfloat16 beside the
        # 143 + 136 times others that are taken away again, 2 * 64 additions of them, each off by up to a step
        bound = h * (16 * R.STEP + EPS[kind] / 2 * 1.01) + TINY[kind]
        if kind == "bfloat16":
            bound = bound + R.gamma(128) * 279 * h.sum(1, keepdims=True)
        want, bound = h[:, np.arange(dim) % hidden], bound[:, np.arange(dim) % hidden]
        close(got[0, TABLE[0, i]:TABLE[0, i + 1]], want, bound + want * EPS[kind] / 2 * 1.01 + TINY[kind], "expert of %d rows" % ROWS[i])
