"""The bounds that the experts' block is held to let honest roundings through, and no mistake: planted here in the expected values, on the CPU."""
import numpy as np
import pytest
import torch

import expert_bounds as B
from token_util import EPS, TORCH, rounded


def to(kind, v):
    return v.to(TORCH[kind]).double()


def plain(x, w_in, w_out, kind):
    """The block with what it rounds rounded."""
    hidden = w_out.shape[1]
    pre = x @ w_in.T
    h = to(kind, pre[:, :hidden] * torch.sigmoid(pre[:, :hidden]) * pre[:, hidden:])
    return to(kind, h @ w_out.T)


class Four:
    def __init__(self, kind, rows, dim, hidden, group):
        rng = np.random.default_rng(dim + hidden + rows)
        self.kind, self.group = kind, group
        self.x = B.f64(rounded(rng.standard_normal((rows, dim)) + 0.5, kind))
        self.q_in, self.q_out = (torch.from_numpy(rng.integers(0, 16, s)).double() for s in ((2 * hidden, dim), (dim, hidden)))
        s_in = rounded(rng.uniform(0.1, 0.4, (2 * hidden, -(-dim // group))) / np.sqrt(dim), kind)
        s_out = rounded(rng.uniform(-0.4, 0.4, (dim, -(-hidden // group))) / np.sqrt(hidden), kind)
        self.s_in, self.s_out = (B.f64(s)[:, torch.arange(k) // group] for s, k in ((s_in, dim), (s_out, hidden)))
        self.want, self.bound = B.forward_four_bits(self.x, (self.q_in - 8) * self.s_in, self.s_in, (self.q_out - 8) * self.s_out,
                                                    self.s_out, kind, group)

    def result(self, x=None, q_in=None, q_out=None, s_in=None, s_out=None):
        def own(v, name):
            return getattr(self, name) if v is None else v
        return plain(own(x, "x"), (own(q_in, "q_in") - 8) * own(s_in, "s_in"), (own(q_out, "q_out") - 8) * own(s_out, "s_out"), self.kind)

    def holds(self, got):
        try:
            B.hold(got.numpy(), self.want, self.bound, self.kind, "")
            return True
        except AssertionError:
            return False


def zeroed(v, columns):
    v = v.clone()
    v[:, columns] = 0 if v.min() < 0 else 8
    return v


MISTAKES = {
    "a tenth less": lambda c: to(c.kind, c.result() * 0.9),
    "a hundredth less": lambda c: to(c.kind, c.result() * 0.99),
    "the last 8 of dim left out": lambda c: c.result(x=zeroed(c.x, slice(-8, None))),
    "the last 2 of dim left out": lambda c: c.result(x=zeroed(c.x, slice(-2, None))),
    "the last 2 of hidden left out": lambda c: c.result(q_out=zeroed(c.q_out, slice(-2, None))),
    "lowest bits turned over": lambda c: c.result(q_out=torch.from_numpy(c.q_out.numpy().astype(int) ^ 1).double()),
    "the next row's scale": lambda c: c.result(s_in=c.s_in.roll(1, 0)),
    "the next group's scale": lambda c: c.result(s_out=c.s_out.roll(c.group, 1)),
    "fewer bits on the way": lambda c: to(c.kind, plain(to("bfloat16", c.x), to("bfloat16", (c.q_in - 8) * c.s_in),
                                                        to("bfloat16", (c.q_out - 8) * c.s_out), "bfloat16")),
}


@pytest.mark.parametrize("kind", ["bfloat16", "half", "float"])
@pytest.mark.parametrize("rows", [33, 130])
@pytest.mark.parametrize("dim,hidden,group", [(776, 328, 32), (384, 1032, 128), (520, 264, 64), (129, 70, 32)])
def test_four_bits(kind, rows, dim, hidden, group):
    c = Four(kind, rows, dim, hidden, group)
    assert c.holds(c.result())
    for name, mistake in MISTAKES.items():
        if name == "fewer bits on the way" and kind == "bfloat16":
            continue
        if name == "the next group's scale" and hidden <= group:
            continue
        if name == "a hundredth less" and kind == "bfloat16":
            continue    # (less than a step and a half of its elements)
        assert not c.holds(mistake(c)), name


@pytest.mark.parametrize("kind", ["bfloat16", "half", "float"])
def test_block(kind):
    """The same for the block of whole weights and its gradients."""
    rng = np.random.default_rng(1)
    n, dim, hidden = 65, 264, 136
    x, dout, w_in, w_out = (B.f64(rounded(rng.standard_normal(s) * scale, kind)) for s, scale in (
        ((n, dim), 1), ((n, dim), 0.5), ((2 * hidden, dim), 1 / 16), ((dim, hidden), 1 / 12)))
    (pre, pre_bound), (out, bound) = B.forward(x, w_in, w_out, kind)
    B.hold(to(kind, pre).numpy(), pre, pre_bound, kind, "")
    B.hold(plain(x, w_in, w_out, kind).numpy(), out, bound, kind, "")
    kept = to(kind, pre)
    grads = B.backward(dout, x, kept, w_in, w_out, kind)
    gate, up, s = kept[:, :hidden], kept[:, hidden:], torch.sigmoid(kept[:, :hidden])
    dh = dout @ w_out
    dpre, h = to(kind, torch.cat([dh * up * (s + gate * s * (1 - s)), dh * gate * s], 1)), to(kind, gate * s * up)
    honest = [dpre @ w_in, dpre.T @ x, dout.T @ h]
    last = zeroed(dpre, slice(-2, None)), zeroed(h, slice(-2, None))
    wrong = [last[0] @ w_in, dpre[:-1].T @ x[:-1], dout[:-1].T @ h[:-1]]
    for good, bad, (want, limit) in zip(honest, wrong, grads):
        B.hold(to(kind, good).numpy(), want, limit, kind, "")
        with pytest.raises(AssertionError):
            B.hold(to(kind, bad).numpy(), want, limit, kind, "")
    with pytest.raises(AssertionError):
        B.hold(plain(zeroed(x, slice(-2, None)), w_in, w_out, kind).numpy(), out, bound, kind, "")
