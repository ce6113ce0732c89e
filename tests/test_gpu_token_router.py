"""Router: experts, gates, counts, balance loss, their gradients and the shuffle's tables, against 64 bits."""
import numpy as np
import pytest

import token_reference as R
from gpu_util import note, runtime
from nvshmem_amd import hip
from token_util import Arrays, EPS, TINY, close, rounded

pytestmark = pytest.mark.gpu

LOWEST = {"float": -3.4028234663852886e38, "half": -65504.0, "bfloat16": -3.3895313892515355e38}


def _logits(rng, kind, shape, how):
    x = rng.standard_normal(shape) * 2
    if how == "ties":          # a few values only, zeros of both signs among them
        x = np.round(x).clip(-2, 2)
        x[rng.random(shape) < 0.3] = -0.0
    if how == "masked":        # single experts, whole tokens, and all experts but one
        npes, tokens, experts = shape
        x[rng.random(shape) < 0.4] = -np.inf
        x[rng.random(shape) < 0.1] = np.nan
        x[rng.random(shape) < 0.1] = LOWEST[kind]
        x[:, tokens // 2] = -np.inf
        x[0, tokens // 3] = np.nan
        x[-1, tokens - 1, 1:] = -np.inf
        x[0, 0] = LOWEST[kind]
    if how == "far":           # far apart, and infinities
        x = x * 20
        x[0, 0, ::3] = np.inf
        x[-1, -1, -1] = np.inf
    return rounded(x, kind)


def _exp_tolerance(logits):
    """What a softmax weight is off by at most, relative, in units of STEP: l - m is rounded once, its product with log2 e
    twice (the constant too) - each of them moves the exponential by as much of |l - m| -, and the exponential is good to two
    steps; the sum of up to 1024 of them goes over at most 16 + 6 additions, its reciprocal and the products with it and with
    the scale take 6 more.  Terms further than 104 away are 0."""
    ok = R.live(logits)
    with np.errstate(invalid="ignore"):
        x = np.where(ok & np.isfinite(logits), logits.astype(np.float64), np.nan)
        far = np.nanmax(x) - np.nanmin(np.where(x >= np.nanmax(x) - 220, x, np.nan)) if np.isfinite(x).any() else 0.0
    return 2 * (3 * min(far, 104.0) + 4) + 22 + 6


SIZES = [  # npes, tokens, experts, topk, shift of the logits in elements
    (8, 37, 256, 8, 0), (4, 5, 64, 4, 0), (16, 9, 176, 6, 1), (1, 3, 1, 1, 0), (3, 20, 33, 16, 3), (2, 70, 1024, 8, 0),
    (4, 11, 300, 2, 1), (8, 1, 8, 1, 0), (2, 90, 60, 5, 2), (4, 40, 256, 10, 0), (2, 6, 513, 16, 0)]


@pytest.mark.parametrize("how", ["normal", "ties", "masked", "far"])
@pytest.mark.parametrize("npes,tokens,experts,topk,shift", SIZES)
@pytest.mark.parametrize("kind", ["float", "half", "bfloat16"])
def test_route(kind, npes, tokens, experts, topk, shift, how):
    rng = np.random.default_rng(experts + tokens)
    x = _logits(rng, kind, (npes, tokens, experts), how)
    tol = _exp_tolerance(x)
    with runtime(npes, 32 << 20) as rt, Arrays(rt) as new:
        logits = new(kind, (tokens, experts), x, shift)
        expert, gate, counts = new("int32", (tokens, topk)), new("float", (tokens, topk)), new("int64", (experts,))
        loss, balance = new("float", (1,)), new("float", (experts,))
        ws = new.workspace("moe_route", tokens, experts)
        for normalise, scale, with_loss in ((True, 1.0, True), (False, 2.5, True), (True, 0.5, False), (False, 1.0, False)):
            note("moe_route", kind, npes, tokens, experts, topk, how, normalise, with_loss)
            for a in (expert, gate, counts, loss, balance):
                a.put(np.array(77).astype(np.float32))
            rt.moe_route(kind, expert.address, gate.address, counts.address, ws.address, logits.address, tokens, experts, topk,
                         loss.address if with_loss else None, balance.address if with_loss else None, normalise, scale)
            rt.sync()
            want_expert, want_gate, want_counts, want_loss, want_balance = R.route(x, topk, normalise, scale)
            assert np.array_equal(expert.get(), want_expert)
            assert np.array_equal(counts.get(), want_counts)
            close(gate.get(), want_gate, tol * R.STEP * want_gate + 1e-37, "gate")
            if with_loss:
                close(balance.get(), np.broadcast_to(want_balance, (npes, experts)), 1.01 * R.STEP * want_balance, "balance")
                # probabilities add up to at most 64 a lane and 8 more in fp32 before 64 bits take over
                close(loss.get(), np.full((npes, 1), want_loss), (tol + 72) * R.STEP * want_loss + 1e-37, "loss")
            else:
                assert (loss.get() == 77).all() and (balance.get() == 77).all()
            ws.get()


@pytest.mark.parametrize("experts", [12, 200, 600])
@pytest.mark.parametrize("kind,nans", [("float", [0x7F800001, 0xFF800001, 0x7FFFFFFF, 0xFFC00000]), ("half", [0x7C01, 0xFC01, 0x7FFF, 0xFE00]),
                                       ("bfloat16", [0x7F81, 0xFF81, 0x7FFF, 0xFFC0])])
def test_every_nan_masks(kind, nans, experts):
    """Signalling and quiet ones of both signs."""
    npes, tokens, topk = 2, 9, 4
    rng = np.random.default_rng(12)
    x = rounded(rng.standard_normal((npes, tokens, experts)), kind)
    at = rng.random(x.shape) < 0.3
    at[0, 0] = True
    bits = np.uint32 if kind == "float" else np.uint16
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        logits, dlogits = new(kind, (tokens, experts), x), new(kind, (tokens, experts))
        for pe in range(npes):
            raw = rt.download(logits.base, pe, (tokens, experts), bits, logits.first)
            raw[at[pe]] = rng.choice(np.array(nans, bits), at[pe].sum())
            rt.upload(logits.base, pe, raw, logits.first)
        x[at] = np.nan
        expert, gate, counts = new("int32", (tokens, topk)), new("float", (tokens, topk)), new("int64", (experts,))
        loss, balance, dloss = new("float", (1,)), new("float", (experts,)), new("float", (1,), np.float32(1))
        ws = new.workspace("moe_route", tokens, experts)
        for normalise in (True, False):
            rt.moe_route(kind, expert.address, gate.address, counts.address, ws.address, logits.address, tokens, experts, topk,
                         loss.address, balance.address, normalise)
            rt.moe_route_grad(kind, dlogits.address, logits.address, expert.address, gate.address, tokens, experts, topk,
                              balance.address, dloss.address, normalise)
            rt.sync()
            want_expert, want_gate, want_counts, want_loss, b = R.route(x, topk, normalise, 1.0)
            tol = _exp_tolerance(x)
            assert np.array_equal(expert.get(), want_expert) and np.array_equal(counts.get(), want_counts)
            close(gate.get(), want_gate, tol * R.STEP * want_gate + 1e-37, "gate")
            close(loss.get(), np.full((npes, 1), want_loss), (tol + 72) * R.STEP * want_loss, "loss")
            want, size = R.route_grad(x, want_expert, gate.get(), balance.get(), np.ones(npes), normalise, 1.0)
            close(dlogits.get(), want, (3 * tol + 52) * R.STEP * size + EPS[kind] / 2 * np.abs(want) * 1.01 + TINY[kind] + 1e-36, "dlogits")


@pytest.mark.parametrize("npes,tokens,experts,topk", [(8, 2100, 256, 8), (2, 17000, 64, 2), (4, 1500, 1024, 3), (8, 0, 16, 2)])
def test_many_tokens_and_none(npes, tokens, experts, topk):
    rng = np.random.default_rng(tokens)
    x = rounded(rng.standard_normal((npes, tokens, experts)) * 2, "bfloat16")
    x[:, tokens - tokens // 16:] = -np.inf
    with runtime(npes, 256 << 20) as rt, Arrays(rt) as new:
        logits = new("bfloat16", (tokens, experts), x)
        expert, gate, counts = new("int32", (tokens, topk)), new("float", (tokens, topk)), new("int64", (experts,))
        loss, balance = new("float", (1,)), new("float", (experts,))
        ws = new.workspace("moe_route", tokens, experts)
        note("moe_route", npes, tokens, experts, topk)
        rt.moe_route("bfloat16", expert.address, gate.address, counts.address, ws.address, logits.address, tokens, experts, topk,
                     loss.address, balance.address)
        rt.sync()
        p = R.softmax(x)
        ok = R.live(x).any(2)
        order = np.argsort(-np.where(R.live(x), x, -np.inf), axis=2, kind="stable")[..., :topk]
        want = np.where(ok[..., None], order, -1)
        got = expert.get()
        assert np.array_equal(got, want)
        want_counts = np.stack([np.bincount(want[pe][want[pe] >= 0], minlength=experts) for pe in range(npes)])
        assert np.array_equal(counts.get(), want_counts)
        c, n = want_counts.sum(0), ok.sum()
        b = experts * c / max(1.0, float(c.sum()) * n)
        want_loss = (b * p.sum((0, 1))).sum()
        close(balance.get(), np.broadcast_to(b, (npes, experts)), 1.01 * R.STEP * b, "balance")
        close(loss.get(), np.full((npes, 1), want_loss), (_exp_tolerance(x) + 72) * R.STEP * want_loss, "loss")
        first = [a.raw() for a in (gate, loss, balance)]
        rt.moe_route("bfloat16", expert.address, gate.address, counts.address, ws.address, logits.address, tokens, experts, topk,
                     loss.address, balance.address)
        rt.sync()
        assert all(np.array_equal(a.raw(), b) for a, b in zip((gate, loss, balance), first)), "the same inputs gave other bits"


@pytest.mark.parametrize("how", ["normal", "ties", "masked", "far"])
@pytest.mark.parametrize("npes,tokens,experts,topk,shift", SIZES)
@pytest.mark.parametrize("kind", ["float", "half", "bfloat16"])
def test_route_grad(kind, npes, tokens, experts, topk, shift, how):
    rng = np.random.default_rng(experts + tokens + 1)
    x = _logits(rng, kind, (npes, tokens, experts), how)
    tol = _exp_tolerance(x)
    want_expert, _, _, _, b = R.route(x, topk, True, 1.0)
    with runtime(npes, 32 << 20) as rt, Arrays(rt) as new:
        dgate_values = rng.standard_normal((npes, tokens, topk)).astype(np.float32)
        up = (1 + np.arange(npes)).astype(np.float32)
        bal = np.broadcast_to(b.astype(np.float32), (npes, experts))
        logits, expert = new(kind, (tokens, experts), x, shift), new("int32", (tokens, topk), want_expert)
        dgate, balance, dloss = new("float", (tokens, topk), dgate_values), new("float", (experts,), bal), new("float", (1,), up[:, None])
        dlogits = new(kind, (tokens, experts), np.float32(9), shift)
        for normalise, scale, with_loss in ((True, 1.0, True), (False, 2.5, True), (True, 0.5, False), (False, 1.0, False)):
            note("moe_route_grad", kind, npes, tokens, experts, topk, how, normalise, with_loss)
            rt.moe_route_grad(kind, dlogits.address, logits.address, expert.address, dgate.address, tokens, experts, topk,
                              balance.address if with_loss else None, dloss.address if with_loss else None, normalise, scale)
            rt.sync()
            want, size = R.route_grad(x, want_expert, dgate_values, bal if with_loss else None, up, normalise, scale)
            # each of the terms holds up to three softmax weights, and sums of up to 1024 products over 22 additions
            close(dlogits.get(), want, (3 * tol + 2 * 22 + 8) * R.STEP * size + EPS[kind] / 2 * np.abs(want) * 1.01 + TINY[kind] + 1e-36,
                  "dlogits")
            assert (dlogits.get()[~R.live(x)] == 0).all()


@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("kind,experts", [("float", 10), ("half", 130), ("bfloat16", 515)])
def test_masked_logits_get_no_gradient_whatever_comes_from_above(kind, experts, normalise):
    npes, tokens, topk = 2, 11, 3
    rng = np.random.default_rng(experts)
    x = rounded(rng.standard_normal((npes, tokens, experts)), kind)
    masked = rng.random(x.shape) < 0.4
    masked[0, 0] = True
    x[masked] = -np.inf
    want_expert, gate, _, _, balance_values = R.route(x, topk, normalise, 1.0)
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        logits, dlogits, expert = new(kind, (tokens, experts), x), new(kind, (tokens, experts)), new("int32", (tokens, topk), want_expert)
        for loss, bad in ((1.0, np.nan), (1.0, np.inf), (np.inf, 1.0), (np.nan, 1.0)):
            dgate_values = np.ones(gate.shape, np.float32)
            dgate_values[:, ::2] = bad                      # (every second token's)
            dgate, dloss = new("float", (tokens, topk), dgate_values), new("float", (1,), np.float32(loss))
            balance = new("float", (experts,), balance_values)
            note("moe_route_grad", kind, experts, normalise, loss, bad)
            rt.moe_route_grad(kind, dlogits.address, logits.address, expert.address, dgate.address, tokens, experts, topk,
                              balance.address, dloss.address, normalise)
            rt.sync()
            got = dlogits.get()
            assert (got[masked] == 0).all()
            if loss == 1.0:
                assert np.isfinite(got[:, 1::2]).all()


@pytest.mark.parametrize("normalise", [True, False])
def test_route_grad_by_differences(normalise):
    """The reference's gradient is the derivative of the reference's value, and the kernel's is the reference's."""
    rng = np.random.default_rng(6)
    npes, tokens, experts, topk, scale = 2, 6, 32, 4, 1.5
    x = rounded(rng.standard_normal((npes, tokens, experts)), "float").astype(np.float64)
    x[0, 1, ::2] = -np.inf
    expert, _, _, _, b = R.route(x, topk, normalise, scale)
    dgate, up = rng.standard_normal((npes, tokens, topk)).astype(np.float32), np.array([0.7, -0.3], np.float32)
    bal = np.broadcast_to(b, (npes, experts))
    want, size = R.route_grad(x, expert, dgate, bal, up, normalise, scale)
    h = 1e-6
    for _ in range(40):
        at = rng.integers(npes), rng.integers(tokens), rng.integers(experts)
        if np.isfinite(x[at]):
            y = [x.copy(), x.copy()]
            y[0][at] += h
            y[1][at] -= h
            slope = (R.route_value(y[0], expert, dgate, bal, up, normalise, scale)
                     - R.route_value(y[1], expert, dgate, bal, up, normalise, scale)) / (2 * h)
            # the value is of the order of 10: differences of it are good to 1e-15 * 10 / h, the step's own error is h^2
            assert abs(slope - want[at]) < 1e-7
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        logits, e, g = new("float", x.shape[1:], x), new("int32", (tokens, topk), expert), new("float", (tokens, topk), dgate)
        balance, dloss, dlogits = new("float", (experts,), bal), new("float", (1,), up[:, None]), new("float", x.shape[1:])
        rt.moe_route_grad("float", dlogits.address, logits.address, e.address, g.address, tokens, experts, topk, balance.address,
                          dloss.address, normalise, scale)
        rt.sync()
        close(dlogits.get(), want, (3 * _exp_tolerance(x) + 52) * R.STEP * size + 1e-36, "dlogits")


def test_route_grad_without_experts_of_its_own():
    """Entries outside the experts count as none, also where the list is not a router's."""
    npes, tokens, experts, topk = 2, 3, 20, 3
    rng = np.random.default_rng(7)
    x = rounded(rng.standard_normal((npes, tokens, experts)) * 3, "half")
    x[0, 2, 4] = -np.inf
    expert = np.array([[19, -1, 20], [1 << 30, 0, -(1 << 31)], [4, 5, -7]], np.int32)
    dgate_values = rng.standard_normal((npes, tokens, topk)).astype(np.float32)
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        logits, e, dgate = new("half", (tokens, experts), x), new("int32", (tokens, topk), expert), new("float", (tokens, topk), dgate_values)
        dlogits = new("half", (tokens, experts))
        clean = np.broadcast_to(np.where((expert >= 0) & (expert < experts), expert, -1), (npes, tokens, topk))
        for normalise in (True, False):
            rt.moe_route_grad("half", dlogits.address, logits.address, e.address, dgate.address, tokens, experts, topk,
                              normalise=normalise)
            rt.sync()
            want, size = R.route_grad(x, clean, dgate_values, None, None, normalise, 1.0)
            close(dlogits.get(), want, (3 * _exp_tolerance(x) + 52) * R.STEP * size + EPS["half"] / 2 * np.abs(want) * 1.01 + TINY["half"],
                  "dlogits")


@pytest.mark.parametrize("cap", [1 << 40, 40, 3, 0])
@pytest.mark.parametrize("npes,tokens,experts,topk", [(8, 37, 256, 8), (4, 5, 4, 1), (2, 700, 64, 16), (16, 33, 176, 6), (3, 50, 3, 2),
                                                      (1, 30, 7, 3), (4, 2049, 8, 4), (2, 20, 1024, 2), (8, 0, 8, 1)])
def test_place(npes, tokens, experts, topk, cap):
    rng = np.random.default_rng(experts)
    e = np.stack([[rng.permutation(experts)[:topk] for _ in range(tokens)] for _ in range(npes)]).reshape(npes, tokens, topk)
    e = np.where(rng.random(e.shape) < 0.1, -1, e).astype(np.int32)
    counts_values = np.stack([np.bincount(e[pe][e[pe] >= 0], minlength=experts) for pe in range(npes)])
    with runtime(npes, 32 << 20) as rt, Arrays(rt) as new:
        expert, counts = new("int32", (tokens, topk), e), new("int64", (experts,), counts_values)
        dest_pe, dest_row = new("int32", (tokens, topk)), new("int64", (tokens, topk))
        expected, expert_row = new("int64", (npes,)), new("int64", (experts // npes + 1,))
        ws = new.workspace("moe_place", tokens, topk, experts)
        note("moe_place", npes, tokens, experts, topk, cap)
        rt.moe_place(dest_pe.address, dest_row.address, expected.address, expert_row.address, ws.address, expert.address,
                     counts.address, tokens, topk, experts, cap)
        rt.sync()
        for got, want in zip((dest_pe, dest_row, expected, expert_row), R.place(e, experts, cap)):
            assert np.array_equal(got.get(), want)
        ws.get()


@pytest.mark.parametrize("npes,tokens,experts,topk", [(2, 66000, 6, 2), (4, 30000, 1024, 4), (8, 20000, 64, 8)])
def test_place_many(npes, tokens, experts, topk):
    """Copies of several blocks, on either side of where a thread takes more of them."""
    rng = np.random.default_rng(tokens)
    e = np.argsort(rng.random((npes, tokens, experts), np.float32) if experts < 100 else rng.random((npes, tokens, 8), np.float32),
                   axis=2)[..., :topk].astype(np.int32)
    if experts >= 100:
        e += 8 * rng.integers(0, experts // 8, (npes, tokens, 1), np.int32)
    e[rng.random(e.shape) < 0.1] = -1
    cap = tokens * topk * 9 // 10
    counts_values = np.stack([np.bincount(e[pe][e[pe] >= 0], minlength=experts) for pe in range(npes)])
    per_pe = experts // npes
    source = np.broadcast_to(np.arange(npes)[:, None, None], e.shape)
    key = np.where(e >= 0, e * npes + source, experts * npes).reshape(-1)
    rank = np.empty(key.size, np.int64)
    rank[np.argsort(key, kind="stable")] = np.arange(key.size)
    first = np.searchsorted(np.sort(key), np.arange(npes + 1) * per_pe * npes)
    pe = np.minimum(key // (per_pe * npes), npes)
    row = rank - first[pe]
    ok = (pe < npes) & (row < cap)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        expert, counts = new("int32", (tokens, topk), e), new("int64", (experts,), counts_values)
        dest_pe, dest_row = new("int32", (tokens, topk)), new("int64", (tokens, topk))
        expected, expert_row = new("int64", (npes,)), new("int64", (per_pe + 1,))
        ws = new.workspace("moe_place", tokens, topk, experts)
        note("moe_place", npes, tokens, experts, topk)
        rt.moe_place(dest_pe.address, dest_row.address, expected.address, expert_row.address, ws.address, expert.address,
                     counts.address, tokens, topk, experts, cap)
        rt.sync()
        assert np.array_equal(dest_pe.get().reshape(-1), np.where(ok, pe, -1))
        assert np.array_equal(dest_row.get().reshape(-1), np.where(ok, row, -1))
        want = np.zeros((npes, npes), np.int64)
        np.add.at(want, (pe[ok], source.reshape(-1)[ok]), 1)
        assert np.array_equal(expected.get(), want)
        ws.get()


def test_place_of_counts_that_are_not_the_experts():
    """Rows may then be given twice, but never outside of what there is."""
    npes, tokens, experts, topk, cap = 4, 300, 16, 2, 50
    rng = np.random.default_rng(8)
    e = rng.integers(-3, experts + 3, (npes, tokens, topk)).astype(np.int32)
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        expert = new("int32", (tokens, topk), e)
        counts = new("int64", (experts,), rng.integers(-(1 << 60), 1 << 60, (npes, experts)))
        dest_pe, dest_row = new("int32", (tokens, topk)), new("int64", (tokens, topk))
        expected, expert_row = new("int64", (npes,)), new("int64", (experts // npes + 1,))
        ws = new.workspace("moe_place", tokens, topk, experts)
        rt.moe_place(dest_pe.address, dest_row.address, expected.address, expert_row.address, ws.address, expert.address,
                     counts.address, tokens, topk, experts, cap)
        rt.sync()
        pe, row = dest_pe.get(), dest_row.get()
        assert ((pe == -1) == (row == -1)).all() and (row < cap).all() and (row >= -1).all()
        assert (pe[pe >= 0] == (e // (experts // npes))[pe >= 0]).all() and (pe[(e < 0) | (e >= experts)] == -1).all()
        ws.get()


def test_in_a_graph_and_on_another_stream():
    rng = np.random.default_rng(10)
    npes, tokens, experts, topk, cap = 4, 90, 64, 4, 130
    with runtime(npes, 32 << 20) as rt, Arrays(rt) as new:
        logits, dlogits = new("float", (tokens, experts)), new("float", (tokens, experts))
        expert, gate, counts = new("int32", (tokens, topk)), new("float", (tokens, topk)), new("int64", (experts,))
        loss, balance, dloss = new("float", (1,)), new("float", (experts,)), new("float", (1,), np.float32(0.5))
        dest_pe, dest_row = new("int32", (tokens, topk)), new("int64", (tokens, topk))
        expected, expert_row = new("int64", (npes,)), new("int64", (experts // npes + 1,))
        ws, ws2 = new.workspace("moe_route", tokens, experts), new.workspace("moe_place", tokens, topk, experts)
        stream = hip.Stream()

        def calls():
            rt.moe_route("float", expert.address, gate.address, counts.address, ws.address, logits.address, tokens, experts, topk,
                         loss.address, balance.address, stream=stream)
            rt.moe_place(dest_pe.address, dest_row.address, expected.address, expert_row.address, ws2.address, expert.address,
                         counts.address, tokens, topk, experts, cap, stream=stream)
            rt.moe_route_grad("float", dlogits.address, logits.address, expert.address, gate.address, tokens, experts, topk,
                              balance.address, dloss.address, stream=stream)

        with hip.Graph(stream) as graph:
            calls()
        for turn in range(4):
            x = _logits(rng, "float", (npes, tokens, experts), ("normal", "ties", "masked", "normal")[turn])
            logits.put(x)
            want_expert, want_gate, want_counts, want_loss, b = R.route(x, topk, True, 1.0)
            seen = []
            for run in (graph.launch, calls):
                for a in (expert, gate, counts, loss, balance, dest_pe, dest_row, dlogits):
                    a.put(np.float32(5))
                hip.synchronize()
                run()
                stream.synchronize()
                assert np.array_equal(expert.get(), want_expert) and np.array_equal(counts.get(), want_counts)
                for got, want in zip((dest_pe, dest_row, expected, expert_row), R.place(want_expert, experts, cap)):
                    assert np.array_equal(got.get(), want)
                seen.append([a.raw() for a in (gate, loss, balance, dlogits)])
            assert all(np.array_equal(a, b) for a, b in zip(*seen))
            close(gate.get(), want_gate, _exp_tolerance(x) * R.STEP * want_gate + 1e-37, "gate")
        graph.destroy()
        stream.destroy()
