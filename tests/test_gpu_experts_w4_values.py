"""The experts' block with weights of 4 bits against 64 bits, within bounds that leave no room for a wrong element."""
import numpy as np
import pytest

import expert_bounds as B
import expert_forms as F
from four_bit_util import ROWS, TABLE, call, values
from gpu_util import runtime
from token_util import Arrays, rounded

pytestmark = pytest.mark.gpu


def operands(rng, kind, npes, mine, dim, hidden, group):
    q_in, q_out = rng.integers(0, 16, (npes, mine, 2 * hidden, dim)), rng.integers(0, 16, (npes, mine, dim, hidden))
    s_in = rng.uniform(0.1, 0.4, (npes, mine, 2 * hidden, -(-dim // group))) / np.sqrt(dim)
    s_out = rng.uniform(-0.4, 0.4, (npes, mine, dim, -(-hidden // group))) / np.sqrt(hidden)
    return q_in, rounded(s_in, kind), q_out, rounded(s_out, kind)


def expected(x, q_in, s_in, q_out, s_out, kind, group):
    def scales(s, k):
        return B.f64(s.astype(np.float64)[:, np.arange(k) // group])
    return B.forward_four_bits(B.f64(x), B.f64(values(q_in, s_in, group)), scales(s_in, x.shape[1]),
                               B.f64(values(q_out, s_out, group)), scales(s_out, q_out.shape[1]), kind, group)


@pytest.mark.parametrize("kind", F.KINDS)
@pytest.mark.parametrize("name,rows,dim,hidden,group", F.FOUR_BIT_CALLS, ids=[c[0] for c in F.FOUR_BIT_CALLS])
def test_every_form(kind, name, rows, dim, hidden, group):
    npes, mine, cap = F.NPES, F.FOUR_BIT_MINE, rows * F.FOUR_BIT_MINE
    rng = np.random.default_rng(rows * dim + group)
    table = F.table(rng, npes, mine, cap, F.FOUR_BIT_ROWS)
    x = np.full((npes, cap, dim), np.nan, np.float32)
    for pe in range(npes):
        x[pe, :table[pe, -1]] = rounded(rng.standard_normal((table[pe, -1], dim)) + 0.5, kind)
    w = operands(rng, kind, npes, mine, dim, hidden, group)
    with runtime(npes, 128 << 20) as rt, Arrays(rt) as new:
        got = call(rt, new, kind, x, *w, table, group)
    for pe in range(npes):
        for i in range(mine):
            a, b = table[pe, i:i + 2]
            if a < b:
                want, bound = expected(x[pe, a:b], *[v[pe, i] for v in w], kind, group)
                B.hold(got[pe, a:b], want, bound, kind, "expert %d of PE %d, %d rows" % (i, pe, b - a))


@pytest.mark.parametrize("kind", F.KINDS)
@pytest.mark.parametrize("group", [32, 64, 96, 128, 384])
@pytest.mark.parametrize("dim,hidden", [(776, 328), (384, 1032), (129, 70), (520, 264)])
def test_long_rows(kind, group, dim, hidden):
    mine, cap = len(ROWS), int(TABLE[0, -1])
    rng = np.random.default_rng(dim + group)
    x = rounded(rng.standard_normal((1, cap, dim)) + 0.5, kind)
    w = operands(rng, kind, 1, mine, dim, hidden, group)
    with runtime(1, 128 << 20) as rt, Arrays(rt) as new:
        got = call(rt, new, kind, x, *w, TABLE, group)
    for i in range(mine):
        a, b = TABLE[0, i:i + 2]
        want, bound = expected(x[0, a:b], *[v[0, i] for v in w], kind, group)
        B.hold(got[0, a:b], want, bound, kind, "expert of %d rows" % (b - a))


def few_places(rng, n, k):
    """A [n, k] of ones and zeros: three ones a row, over all rows in every place where there are rows enough, at the ends in all experts."""
    on = np.zeros((n, k), bool)
    at = np.arange(n)
    on[at, 2 * at % k] = on[at, (2 * at + 1) % k] = True
    on[at, np.where(at % 3 == 0, k - 1, np.where(at % 3 == 1, 0, rng.integers(0, k, n)))] = True
    return on


@pytest.mark.parametrize("kind", F.KINDS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dim,hidden", [(520, 264), (263, 330), (65536, 8), (8, 65536)])
def test_few_products(kind, group, dim, hidden):
    """Rows, and weights of the second product, with three elements that are not zero, at the ends of rows and all over them: a product that is
    left out, has another's scale or lost bits of its element is far outside the bounds."""
    rows = [1, 40, 129] if dim * hidden > 300000 else ROWS
    table = np.concatenate([[0], np.cumsum(rows)])[None]
    mine, cap = len(rows), int(table[0, -1])
    rng = np.random.default_rng(dim + group)
    x = np.where(few_places(rng, cap, dim), rounded(rng.uniform(0.5, 2, (cap, dim)) * rng.choice([-1, 1], (cap, dim)), kind), 0)[None].astype(np.float32)
    q_in, s_in, q_out, s_out = operands(rng, kind, 1, mine, dim, hidden, group)
    s_in, s_out = rounded(s_in * np.sqrt(dim), kind), rounded(s_out * np.sqrt(hidden), kind)
    for i in range(mine):
        q_out[0, i] = np.where(few_places(rng, dim, hidden), np.where(q_out[0, i] == 8, 9, q_out[0, i]), 8)
    if hidden == 65536:     # up is zero almost everywhere, and so is h
        kept = np.unique(np.concatenate([[0, 1, 63, 64, 127, 128, 255, 256, 32767, 32768, hidden - 2, hidden - 1], rng.integers(0, hidden, 40)]))
        q_in[0, :, hidden + np.setdiff1d(np.arange(hidden), kept)] = 8
        q_out[0] = rng.integers(0, 16, q_out[0].shape)
    with runtime(1, 512 << 20) as rt, Arrays(rt) as new:
        got = call(rt, new, kind, x, q_in, s_in, q_out, s_out, table, group)
    for i in range(mine):
        a, b = table[0, i:i + 2]
        want, bound = expected(x[0, a:b], q_in[0, i], s_in[0, i], q_out[0, i], s_out[0, i], kind, group)
        B.close(got[0, a:b], want, bound, "expert of %d rows" % (b - a))
