"""The experts' block in 64 bits with bounds as narrow as its kernels' sums allow: what they add is counted, zeros are not.

A matrix core may round each of its additions by up to a whole step of fp32 (2^-23 of what is added); an addition of zero changes nothing.  So a sum
is off by no more than its products that are not zero, and two, times 2^-23 of the sum of their magnitudes.  Sigmoid and what is multiplied
with it are off by 16 half steps, each rounding to the type by half of its step.

Beside the bounds, which take every error at its worst, rms() holds what is off on average to what roundings to the type alone give."""
import numpy as np
import torch

from expert_reference import FEW, STEP, f64
from token_util import EPS, TINY, close


def count(a, b):
    """The products of a b^T that are not zero, for each of its elements."""
    return (a != 0).double() @ (b != 0).double().T


def product(a, da, b):
    """a b^T where a is known to da: the value and what it may be off by."""
    return a @ b.T, da @ b.abs().T + (count(a, b) + 2) * 2 * STEP * ((a.abs() + da) @ b.abs().T)


def rounding(v, kind):
    return torch.where(v == 0, 0.0, v.abs() * (EPS[kind] / 2) * 1.01 + TINY[kind])


def rounded_too(v, dv, kind):
    return torch.where((v == 0) & (dv == 0), 0.0, dv + (v.abs() + dv) * (EPS[kind] / 2) * 1.01 + TINY[kind])


def activation(pre, dpre, hidden, kind):
    """h = silu(gate) * up, as it is rounded on its way to the second product."""
    gate, up, dgate, dup = pre[:, :hidden], pre[:, hidden:], dpre[:, :hidden], dpre[:, hidden:]
    silu = gate * torch.sigmoid(gate)
    dsilu = 1.1 * dgate + FEW * silu.abs()          # (the derivative of silu is at most 1.1)
    h = silu * up
    return h, rounded_too(h, (silu.abs() + dsilu) * (up.abs() + dup) - silu.abs() * up.abs() + STEP * h.abs(), kind)


def forward(x, w_in, w_out, kind):
    """(pre, bound), (out, bound)"""
    pre, dpre = product(x, torch.zeros_like(x), w_in)
    out, dout = product(*activation(pre, dpre, w_out.shape[1], kind), w_out)
    return (pre, dpre + rounding(pre, kind)), (out, rounded_too(out, dout, kind))


def backward(dout, x, pre, w_in, w_out, kind):
    """(drows, bound), (dw_in, bound), (dw_out, bound)"""
    hidden = w_out.shape[1]
    gate, up = pre[:, :hidden], pre[:, hidden:]
    s = torch.sigmoid(gate)
    silu = gate * s
    dh, ddh = product(dout, torch.zeros_like(dout), w_out.T)
    slope, slope_size = s + silu * (1 - s), s + silu.abs() * (1 - s)
    dpre = torch.cat([dh * up * slope, dh * silu], 1)
    ddpre = torch.cat([(ddh * slope.abs() + FEW * (dh.abs() + ddh) * slope_size) * up.abs() * 1.01, ddh * silu.abs() * 1.01 + FEW * (dh * silu).abs()], 1)
    ddpre = rounded_too(dpre, ddpre, kind)
    h = silu * up
    dh_own = rounded_too(h, FEW * h.abs(), kind)
    results = [product(dpre, ddpre, w_in.T), product(dpre.T, ddpre.T, x.T), product(h.T, dh_own.T, dout.T)]
    results = [(v, rounded_too(v, bound, kind)) for v, bound in results]
    return results[0], results[1], (results[2][0].T, results[2][1].T)


def step_of(kind, group, few):
    """k that are added up in front of their scale."""
    if few:
        return 128 if group % 128 == 0 else 64 if group % 64 == 0 else 32
    return 64 if kind != "float" and group % 64 == 0 else 32


def forward_four_bits(x, w_in, s_in, w_out, s_out, kind, group):
    """(out, bound) for weights w = (q - 8) s, s expanded like w.  Within a step products of q - 8 are added up, of an fp32 element of
    experts of up to 64 rows in three parts; of a bfloat16 one of such an expert, first -136 and then 128 + q.  Then the step's sum, times s,
    goes to the others' by one operation."""
    few = x.shape[0] <= 64
    step = step_of(kind, group, few)

    def product4(a, da, w, s):
        k, size = a.shape[1], a.abs() + da
        own = size @ w.abs().T
        if few and kind == "bfloat16":
            added = 2 * (a != 0).double().sum(1, keepdim=True).clamp(max=step)
            magnitude = size @ (279 * s.abs()).T
        else:
            added = (3 if few and kind == "float" else 1) * count(a, w).clamp(max=step)
            magnitude = own * (1 + 2.0 ** -7)
        return a @ w.T, da @ w.abs().T + (added + 2) * 2 * STEP * magnitude + -(-k // step) * STEP * own

    out, dout = product4(*activation(*product4(x, torch.zeros_like(x), w_in, s_in), w_out.shape[1], kind), w_out, s_out)
    return out, rounded_too(out, dout, kind)


def rms_limit(kind, added=386):
    """What is off on average, relative to the result.  Two roundings to the type on the way (h or its gradients, and the result), each of up to half
    a step and even in that: 2^0.5 / 3^0.5 half steps together at the most.  fp32: sums of up to `added` in a row, of which
    additions at half a step each add up where the core cuts off; twice, one product after the other."""
    return EPS[kind] / 2 if kind != "float" else 2 * added * STEP


def rms(got, want):
    got, want = f64(np.asarray(got)), torch.as_tensor(want)
    size = (want ** 2).mean().sqrt()
    return float(((got - want) ** 2).mean().sqrt() / size) if want.numel() and size else 0.0


def hold(got, want, bound, kind, what):
    """Within the bound everywhere, and on average off by no more than roundings are."""
    close(got, want, bound, what)
    assert rms(got, want) <= rms_limit(kind), "%s: off by %.3g of its size, more than %.3g" % (what, rms(got, want), rms_limit(kind))
