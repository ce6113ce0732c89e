"""The experts' block with as many experts as it takes, and dropout on more elements than 32 bits count."""
import numpy as np
import pytest

import expert_bounds as B
from dropout_reference import philox
from four_bit_util import call, values
from gpu_util import note, runtime
from token_util import Arrays, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("npes", [1, 4])
@pytest.mark.parametrize("cap_of_one", [3, 40])     # (tiles of 32 rows, whose blocks have half the wavefronts, and of 128)
def test_1024_experts(npes, cap_of_one):
    kind, mine, dim, hidden, group = "bfloat16", 1024 // npes, 24, 16, 32
    cap = cap_of_one * mine
    rng = np.random.default_rng(npes + cap_of_one)
    sizes = rng.choice([0, 0, 1, 2, 5], (npes, mine))
    sizes[:, -1], sizes[:, 0], sizes[0, mine // 2] = 2, 1, 70
    table = np.concatenate([np.zeros((npes, 1), np.int64), np.cumsum(sizes, 1)], 1)
    assert table.max() <= cap
    x, dout = (np.full((npes, cap, dim), np.nan, np.float32) for _ in range(2))
    pre = np.full((npes, cap, 2 * hidden), np.nan, np.float32)
    for pe in range(npes):
        for a in (x, dout, pre):
            a[pe, :table[pe, -1]] = rounded(rng.standard_normal((table[pe, -1], a.shape[2])), kind)
    w_in, w_out = (rounded(rng.standard_normal((npes, mine) + s) / 4, kind) for s in ((2 * hidden, dim), (dim, hidden)))
    q_in, q_out = rng.integers(0, 16, w_in.shape), rng.integers(0, 16, w_out.shape)
    s_in, s_out = (rounded(rng.uniform(0.01, 0.1, w.shape[:3] + (1,)), kind) for w in (w_in, w_out))
    with runtime(npes, 128 << 20) as rt, Arrays(rt) as new:
        er, xa, da, pa, wi, wo = (new(k, v.shape[1:], v) for k, v in (("int64", table), (kind, x), (kind, dout), (kind, pre), (kind, w_in), (kind, w_out)))
        out, drows, dw_in, dw_out = (new(kind, v.shape[1:]) for v in (x, x, w_in, w_out))
        ws = new.workspace("moe_experts_grad", cap, 1024, dim, hidden)
        note("1024 experts", npes, cap)
        rt.moe_experts(kind, out.address, ws.address, xa.address, wi.address, wo.address, er.address, cap, 1024, dim, hidden)
        rt.moe_experts_grad(kind, drows.address, dw_in.address, dw_out.address, ws.address, da.address, xa.address, pa.address, wi.address,
                            wo.address, er.address, cap, 1024, dim, hidden)
        rt.sync()
        four = call(rt, new, kind, x, q_in, s_in, q_out, s_out, table, group)
        out, drows, dw_in, dw_out = (a.get() for a in (out, drows, dw_in, dw_out))
    for pe in range(npes):
        for i in range(mine):
            own = slice(*table[pe, i:i + 2])
            if own.start == own.stop:
                assert not dw_in[pe, i].any() and not dw_out[pe, i].any()
                continue
            w = B.f64(w_in[pe, i]), B.f64(w_out[pe, i])
            want, bound = B.forward(B.f64(x[pe, own]), *w, kind)[1]
            B.close(out[pe, own], want, bound, "out of expert %d" % i)
            grads = B.backward(B.f64(dout[pe, own]), B.f64(x[pe, own]), B.f64(pre[pe, own]), *w, kind)
            for got, (want, bound) in zip((drows[pe, own], dw_in[pe, i], dw_out[pe, i]), grads):
                B.close(got, want, bound, "gradients of expert %d" % i)
            scales = [B.f64(np.broadcast_to(s[pe, i], q[pe, i].shape)) for s, q in ((s_in, q_in), (s_out, q_out))]
            want, bound = B.forward_four_bits(B.f64(x[pe, own]), B.f64(values(q_in[pe, i], s_in[pe, i], group)), scales[0],
                                              B.f64(values(q_out[pe, i], s_out[pe, i], group)), scales[1], kind, group)
            B.close(four[pe, own], want, bound, "4 bits of expert %d" % i)


def test_dropout_beyond_2_32_elements():
    """The last rows of more than 2^32 elements."""
    tokens, dim, p, seed = 600_001, 7168, 0.25, [7, 9]
    elems, limit = tokens * dim, 16384
    assert elems > 1 << 32
    places = [0, (1 << 32) // dim - 1, tokens - 2]       # rows, two at a time
    rng = np.random.default_rng(0)
    with runtime(1, 20 << 30) as rt:
        import torch
        rows, out, s = rt.malloc(elems * 2), rt.malloc(elems * 2), rt.malloc(16)
        rt.upload(s, 0, np.array(seed, np.int64))
        x = {t: torch.from_numpy(rng.standard_normal((2, dim)).astype(np.float32)).to(torch.bfloat16) for t in places}
        for t, v in x.items():
            rt.upload(rows, 0, v.view(torch.int16).numpy(), t * dim * 2)
        note("dropout beyond 2^32")
        rt.dropout("bfloat16", out, rows, s, tokens, dim, p)
        rt.sync()
        for t, v in x.items():
            got = torch.from_numpy(rt.download(out, 0, (2, dim), np.int16, t * dim * 2)).view(torch.bfloat16)
            block = np.arange(t * dim // 8, (t + 2) * dim // 8, dtype=np.uint64)
            zero = np.zeros_like(block)
            words = np.stack(philox([block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), zero + np.uint64(seed[1]), zero], [seed[0], 0]), 1)
            kept = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(2, dim) >= limit
            want = torch.where(torch.from_numpy(kept), (v.double() * (65536 / (65536 - limit))).to(torch.float32).to(torch.bfloat16), torch.zeros_like(v))
            assert torch.equal(got, want), t
