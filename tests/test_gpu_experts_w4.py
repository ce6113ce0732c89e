"""The experts' block with weights of 4 bits against 64 bits."""
import numpy as np
import pytest
import torch

import expert_reference as R
from gpu_util import note, runtime
from test_gpu_experts import KINDS, starts
from token_util import Arrays, close, rounded

pytestmark = pytest.mark.gpu


def packed(new, rng, npes, mine, n, k, shift):
    v = rng.integers(0, 256, (npes, mine, n, (k + 1) // 2)).astype(np.uint8)   # (the last half of a row of an odd k is anything)
    return v, new("byte", v.shape[1:], v, shift)


def check(rt, new, rng, kind, mine, cap, dim, hidden, group, expert_row, shift=0):
    npes = rt.npes
    er = new("int64", (mine + 1,), expert_row)
    busy = np.zeros((npes, cap), bool)
    for pe in range(npes):
        for a, b in R.ranges(expert_row[pe], cap):
            busy[pe, a:b] = True
    x_values = np.where(busy[..., None], rounded(rng.standard_normal((npes, cap, dim)), kind), np.nan).astype(np.float32)
    x = new(kind, (cap, dim), x_values, shift)
    q_in, w_in = packed(new, rng, npes, mine, 2 * hidden, dim, shift)
    q_out, w_out = packed(new, rng, npes, mine, dim, hidden, shift)
    s_in_values = rounded(rng.uniform(0.1, 0.4, (npes, mine, 2 * hidden, -(-dim // group))) / np.sqrt(dim), kind)
    s_out_values = rounded(rng.uniform(-0.4, 0.4, (npes, mine, dim, -(-hidden // group))) / np.sqrt(hidden), kind)
    s_in, s_out = new(kind, s_in_values.shape[1:], s_in_values, shift), new(kind, s_out_values.shape[1:], s_out_values, shift)
    out, ws = new(kind, (cap, dim), None, shift), new.workspace("moe_experts", cap, mine * npes, dim, hidden)
    untouched = out.get()
    note("moe_experts_w4", kind, npes, mine, cap, dim, hidden, group, expert_row.tolist())
    rt.moe_experts_w4(kind, out.address, ws.address, x.address, w_in.address, s_in.address, w_out.address, s_out.address, er.address,
                      cap, mine * npes, dim, hidden, group)
    rt.sync()
    ws.get()
    got = out.get()
    for pe in range(npes):
        for i, (a, b) in enumerate(R.ranges(expert_row[pe], cap)):
            def expand(s, k):
                return R.f64(s)[:, torch.arange(k) // group]
            want, bound = R.forward_four_bits(R.f64(x_values[pe, a:b]), R.four_bits(q_in[pe, i], s_in_values[pe, i], dim, group),
                                              expand(s_in_values[pe, i], dim),
                                              R.four_bits(q_out[pe, i], s_out_values[pe, i], hidden, group),
                                              expand(s_out_values[pe, i], hidden), kind)
            close(got[pe, a:b], want, bound, "out of expert %d of PE %d" % (i, pe))
    assert np.array_equal(got[~busy], untouched[~busy])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group", [32, 64, 128, 96, 384])
@pytest.mark.parametrize("dim,hidden", [(256, 128), (1, 1), (7, 33), (129, 70), (520, 264), (384, 1032)])
def test_sizes(kind, group, dim, hidden):
    npes, mine, cap = 2, 5, 330
    rng = np.random.default_rng(dim * 1000 + hidden + group)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        check(rt, new, rng, kind, mine, cap, dim, hidden, group, starts(npes, mine, cap, [0, 1, 37, 200, 17], rng, 3))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("sizes", [[0], [1], [15, 16, 17], [31, 32, 33], [127, 128, 129], [300, 0, 0, 1]])
def test_rows_of_an_expert(kind, sizes):
    npes, mine, dim, hidden = 3, 4, 136, 200
    rng = np.random.default_rng(sum(sizes) + 1)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        cap = sum(int(v) for v in np.resize(sizes, mine)) + 9
        check(rt, new, rng, kind, mine, cap, dim, hidden, 64, starts(npes, mine, cap, sizes, rng))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shift", [1, 3])
def test_operands_on_any_element(kind, shift):
    npes, mine, cap, dim, hidden = 2, 3, 150, 264, 72
    rng = np.random.default_rng(shift)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        check(rt, new, rng, kind, mine, cap, dim, hidden, 128, starts(npes, mine, cap, [70, 5, 40], rng, 2), shift)


@pytest.mark.parametrize("kind", ["bfloat16", "half"])
@pytest.mark.parametrize("group", [32, 64])
def test_tiles_of_256_rows(kind, group):
    npes, mine, dim, hidden = 2, 3, 776, 328
    rng = np.random.default_rng(group)
    with runtime(npes, 128 << 20) as rt, Arrays(rt) as new:
        check(rt, new, rng, kind, mine, 960, dim, hidden, group, starts(npes, mine, 960, [500, 257, 190], rng, 4))


@pytest.mark.parametrize("npes,mine", [(1, 1), (1, 130), (16, 2), (64, 1)])
def test_numbers_of_pes_and_experts(npes, mine):
    cap, dim, hidden = 200, 48, 40
    rng = np.random.default_rng(npes)
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        check(rt, new, rng, "bfloat16", mine, cap, dim, hidden, 32, starts(npes, mine, cap, [0, 3, 0, 1, 20, 0, 0, 2], rng))


@pytest.mark.parametrize("kind", ["bfloat16", "float"])      # (h is up to 448 * 1025 * 8 with halves, which hold 65504)
def test_large_and_small_elements(kind):
    """One product that is known: weights of -8 to 7 with scale 1 on unit rows come back as they are, on rows of one huge element exactly
    scaled (fp32 elements keep all their bits)."""
    npes, mine, dim, hidden, group, n = 1, 1, 64, 64, 32, 40
    rng = np.random.default_rng(1)
    value = {"float": 16777213.0, "bfloat16": 257.0 / 256}[kind]
    value = float(rounded(np.array([value]), kind)[0])
    x = np.zeros((npes, n, dim), np.float32)
    x[0, np.arange(n), np.arange(n) % dim] = value
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        # gate: every weight is 7 and the scale large, so that gate * sigmoid(gate) is gate; up: the weights in question
        q_in = np.full((1, 1, 2 * hidden, dim // 2), 0xff, np.uint8)
        q_up = rng.integers(0, 16, (hidden, dim))
        q_in[0, 0, hidden:] = q_up[:, 0::2] | q_up[:, 1::2] << 4
        s_in = np.ones((1, 1, 2 * hidden, dim // group), np.float32)
        s_in[0, 0, :hidden] = rounded(np.array([64.0 / value]), kind)[0]
        q_out = np.full((1, 1, dim, hidden // 2), 0x88, np.uint8)
        for i in range(dim):
            q_out[0, 0, i, i // 2] = 0x98 if i % 2 else 0x89     # one in place i, zeros elsewhere
        s_out = np.ones((1, 1, dim, hidden // group), np.float32)
        operands = [new(kind, x.shape[1:], x), new("byte", q_in.shape[1:], q_in), new(kind, s_in.shape[1:], s_in),
                    new("byte", q_out.shape[1:], q_out), new(kind, s_out.shape[1:], s_out), new("int64", (2,), np.array([[0, n]]))]
        out, ws = new(kind, (n, dim)), new.workspace("moe_experts", n, 1, dim, hidden)
        note("known product", kind)
        rt.moe_experts_w4(kind, out.address, ws.address, *[o.address for o in operands], n, 1, dim, hidden, group)
        rt.sync()
        gate = 7 * float(s_in[0, 0, 0, 0]) * value
        want = np.array([[gate * value * (q_up[c, i] - 8) for c in range(dim)] for i in range(n)])
        close(out.get()[0], want, 2 * (np.finfo(np.float32).eps * 8 + R.EPS[kind]) * np.abs(want))
