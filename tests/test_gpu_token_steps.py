"""Batches of which a block or a wavefront takes several steps, on either side of the sizes where shapes switch, against 64 bits."""
import numpy as np
import pytest

import token_reference as R
from gpu_util import note, runtime
from test_gpu_token_router import _exp_tolerance
from token_util import Arrays, EPS, TINY, close, rounded

pytestmark = pytest.mark.gpu

MODES = [(True, 1.0, True), (False, 2.5, True), (True, 0.5, False), (False, 1.0, False)]      # normalise, scale, with the loss


def _logits(rng, kind, shape):
    """Single experts masked, every 97th token, and the last sixteenth of a batch."""
    x = rng.standard_normal(shape) * 2
    x[rng.random(shape) < 0.1] = -np.inf
    x[rng.random(shape) < 0.02] = np.nan
    x[:, ::97] = -np.inf
    x[:, shape[1] - shape[1] // 16:] = -np.inf
    return rounded(x, kind)


@pytest.mark.parametrize("npes,tokens,experts,topk", [(8, 2100, 256, 8), (2, 17000, 64, 2), (4, 1500, 1024, 3), (3, 7000, 40, 12)])
@pytest.mark.parametrize("kind", ["float", "half", "bfloat16"])
def test_router(kind, npes, tokens, experts, topk):
    """Blocks of 1024 threads that take two and three steps."""
    rng = np.random.default_rng(tokens)
    x = _logits(rng, kind, (npes, tokens, experts))
    tol = _exp_tolerance(x)
    with runtime(npes, 128 << 20) as rt, Arrays(rt) as new:
        logits = new(kind, (tokens, experts), x, 1)
        expert, gate, counts = new("int32", (tokens, topk)), new("float", (tokens, topk)), new("int64", (experts,))
        loss, balance = new("float", (1,)), new("float", (experts,))
        ws = new.workspace("moe_route", tokens, experts)
        for normalise, scale, with_loss in MODES:
            note("moe_route", kind, npes, tokens, experts, topk, normalise, with_loss)
            for a in (expert, gate, counts, loss, balance):
                a.put(np.array(77).astype(np.float32))
            rt.moe_route(kind, expert.address, gate.address, counts.address, ws.address, logits.address, tokens, experts, topk,
                         loss.address if with_loss else None, balance.address if with_loss else None, normalise, scale)
            rt.sync()
            want_expert, want_gate, want_counts, want_loss, want_balance = R.route_many(x, topk, normalise, scale)
            assert np.array_equal(expert.get(), want_expert) and np.array_equal(counts.get(), want_counts)
            close(gate.get(), want_gate, tol * R.STEP * want_gate + 1e-37, "gate")
            if with_loss:
                close(balance.get(), np.broadcast_to(want_balance, (npes, experts)), 1.01 * R.STEP * want_balance, "balance")
                # in fp32 a lane adds up at most 64 shares, 2 lanes their sums, 16 wavefronts theirs; the rest is in 64 bits
                close(loss.get(), np.full((npes, 1), want_loss), (tol + 64 + 2 + 16) * R.STEP * want_loss, "loss")
            else:
                assert (loss.get() == 77).all() and (balance.get() == 77).all()
            ws.get()


@pytest.mark.parametrize("npes,tokens,experts,topk", [(1, 1_060_000, 8, 2), (2, 530_001, 6, 3), (2, 140_000, 260, 4)])
def test_router_of_a_million_tokens(npes, tokens, experts, topk):
    """A lane then adds up the most shares that it ever does, and there are as many blocks as that takes."""
    period = 1009
    rng = np.random.default_rng(experts)
    some = _logits(rng, "bfloat16", (npes, period, experts))
    turn = np.arange(tokens) % period
    tol = _exp_tolerance(some)
    want_expert, want_gate, _, _, _ = R.route_many(some, topk, True, 1.0)
    p, ok = R.softmax(some), R.live(some).any(2)
    times = np.bincount(turn, minlength=period)          # how often each of the rows is in the batch
    want_counts = np.zeros((npes, experts), np.int64)
    for pe in range(npes):
        np.add.at(want_counts[pe], want_expert[pe][want_expert[pe] >= 0],
                  np.broadcast_to(times[:, None], (period, topk))[want_expert[pe] >= 0])
    c, n = want_counts.sum(0), (ok * times).sum()
    b = experts * c / (float(c.sum()) * n)
    want_loss = (b * (p * times[:, None]).sum((0, 1))).sum()
    with runtime(npes, 256 << 20) as rt, Arrays(rt) as new:
        logits = new("bfloat16", (tokens, experts), some[:, turn])
        expert, gate, counts = new("int32", (tokens, topk)), new("float", (tokens, topk)), new("int64", (experts,))
        loss, balance, ws = new("float", (1,)), new("float", (experts,)), new.workspace("moe_route", tokens, experts)
        note("moe_route", npes, tokens, experts, topk)
        rt.moe_route("bfloat16", expert.address, gate.address, counts.address, ws.address, logits.address, tokens, experts, topk,
                     loss.address, balance.address)
        rt.sync()
        assert np.array_equal(counts.get(), want_counts)
        assert np.array_equal(expert.get(), want_expert[:, turn])
        close(gate.get(), want_gate[:, turn], (tol * R.STEP * want_gate + 1e-37)[:, turn], "gate")
        close(balance.get(), np.broadcast_to(b, (npes, experts)), 1.01 * R.STEP * b, "balance")
        close(loss.get(), np.full((npes, 1), want_loss), (tol + 64 + 2 + 16) * R.STEP * want_loss, "loss")
        ws.get()


@pytest.mark.parametrize("npes,tokens,experts,topk", [(8, 4500, 64, 6), (4, 4300, 200, 8), (2, 4200, 300, 4), (1, 4300, 1024, 1)])
@pytest.mark.parametrize("kind", ["float", "half", "bfloat16"])
def test_router_gradient(kind, npes, tokens, experts, topk):
    """Two to three steps a block, the last one ragged.  Its table of what only the chosen experts get goes from one token to the
    next: the same tokens in calls of one step a block have the same bits."""
    rng = np.random.default_rng(tokens + 1)
    x = _logits(rng, kind, (npes, tokens, experts))
    tol = _exp_tolerance(x)
    with runtime(npes, 128 << 20) as rt, Arrays(rt) as new:
        up = (1 + np.arange(npes)).astype(np.float32)
        dgate_values = rng.standard_normal((npes, tokens, topk)).astype(np.float32)
        want_expert, _, _, _, b = R.route_many(x, topk, True, 1.0)
        bal = np.broadcast_to(b.astype(np.float32), (npes, experts))
        logits, expert = new(kind, (tokens, experts), x, 1), new("int32", (tokens, topk), want_expert)
        dgate, balance, dloss = new("float", (tokens, topk), dgate_values), new("float", (experts,), bal), new("float", (1,), up[:, None])
        dlogits, parts = new(kind, (tokens, experts), np.float32(9), 1), new(kind, (tokens, experts), np.float32(9), 1)
        size = 4 if kind == "float" else 2
        step = 1024 // npes * (256 // (16 if experts <= 256 else 64))         # tokens of one step of all of a PE's blocks
        assert tokens > step
        for normalise, scale, with_loss in MODES:
            more = dict(balance=balance.address, dloss=dloss.address) if with_loss else {}
            note("moe_route_grad", kind, npes, tokens, experts, topk, normalise, with_loss)
            rt.moe_route_grad(kind, dlogits.address, logits.address, expert.address, dgate.address, tokens, experts, topk,
                              normalise=normalise, scale=scale, **more)
            for t in range(0, tokens, step):
                rt.moe_route_grad(kind, parts.address + t * experts * size, logits.address + t * experts * size,
                                  expert.address + t * topk * 4, dgate.address + t * topk * 4, min(step, tokens - t), experts, topk,
                                  normalise=normalise, scale=scale, **more)
            rt.sync()
            got = dlogits.get()
            assert np.array_equal(got, parts.get())
            want, magnitude = R.route_grad_many(x, want_expert, dgate_values, bal if with_loss else None, up, normalise, scale)
            # each of the terms holds up to three softmax weights, and sums of up to 1024 products over 22 additions
            close(got, want, (3 * tol + 2 * 22 + 8) * R.STEP * magnitude + EPS[kind] / 2 * np.abs(want) * 1.01 + TINY[kind] + 1e-36,
                  "dlogits")
            assert (got[~R.live(x)] == 0).all()


@pytest.mark.parametrize("npes,tokens", [(1, 12288), (1, 12289), (8, 1536), (8, 1537), (3, 2735), (8, 16384), (8, 16385), (4, 75001)])
@pytest.mark.parametrize("vocab", [300, 511, 512, 70001, 1 << 20])
def test_tables_gradient(npes, tokens, vocab):
    """The most tokens that are sorted by counting, and the fewest that are sorted by digits, by one, two and three of them; and blocks that
    sort one tile of 2048 tokens, two, and three with a ragged last one.  A third of the tokens name one row."""
    rng = np.random.default_rng(tokens)
    rows, dim = -(-vocab // npes), 3
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        ids_values = np.minimum(np.exp(rng.random((npes, tokens)) * np.log(vocab)).astype(np.int64) - 1, vocab - 1)
        ids_values[rng.random((npes, tokens)) < 0.3] = vocab // 2
        ids_values[rng.random((npes, tokens)) < 0.1] = -1
        ids_values[:, ::50] = 1 << 40
        # whole numbers, whose sums of fp32 are exact
        dout_values = rng.integers(-8, 9, (npes, tokens, dim)).astype(np.float32)
        dout, ids = new("float", (tokens, dim), dout_values), new("int64", (tokens,), ids_values)
        dtable, ws = new("float", (rows, dim), np.float32(7)), new.workspace("embedding_grad", tokens, vocab, dim)
        note("embedding_grad", npes, tokens, vocab)
        rt.embedding_grad("float", dtable.address, dout.address, ids.address, ws.address, tokens, vocab, dim, 1.0)
        rt.sync()
        want, _, _ = R.embedding_grad(np.full((npes, rows, dim), 7.0), dout_values, ids_values, vocab, 1.0)
        assert np.array_equal(dtable.get(), want)
        ws.get()


def test_sums_of_more_parts_than_a_grid_has_rows():
    """64 tokens to a part: 65 626 parts, most of them of one row."""
    tokens, vocab, dim = 4_200_010, 7, 2
    rng = np.random.default_rng(1)
    with runtime(1, 256 << 20) as rt, Arrays(rt) as new:
        ids_values = rng.choice(np.array([0, 2, 3, 3, 3, 3, 6, -1]), (1, tokens))
        # ones of both signs, whose sums stay below 2^24
        dout_values = rng.choice(np.array([-1, 1], np.float32), (1, tokens, dim))
        dout, ids = new("float", (tokens, dim), dout_values), new("int64", (tokens,), ids_values)
        dtable, ws = new("float", (vocab, dim), np.float32(7)), new.workspace("embedding_grad", tokens, vocab, dim)
        note("embedding_grad", tokens)
        rt.embedding_grad("float", dtable.address, dout.address, ids.address, ws.address, tokens, vocab, dim, 1.0)
        rt.sync()
        want = [[dout_values[0, ids_values[0] == v, i].sum(dtype=np.float64) for i in range(dim)] for v in range(vocab)]
        assert np.array_equal(dtable.get()[0], want)
        ws.get()


# tokens, dim: wavefronts of a whole row and of shared ones, of one token and of four
@pytest.mark.parametrize("tokens,dim", [(65_600, 1032), (262_160, 264), (525_000, 130), (4_194_400, 3)])
def test_more_rows_than_a_grid_has(tokens, dim):
    """Lookup and sum of one copy, where blocks come round to a second group of tokens."""
    vocab, cap = 50, 40
    rng = np.random.default_rng(dim)
    with runtime(1, 1 << 30) as rt, Arrays(rt) as new:
        table_values = rounded(rng.standard_normal((vocab, dim)), "half")
        table, ids_values = new("half", (vocab, dim), table_values), rng.integers(-1, vocab + 1, (1, tokens))
        ids, out = new("int64", (tokens,), ids_values), new("half", (tokens, dim))
        note("embedding", tokens, dim)
        rt.embedding("half", out.address, table.address, ids.address, tokens, vocab, dim, 1.0)
        rt.sync()
        with_zeros = np.concatenate([table_values, np.zeros((1, dim), np.float32)])
        assert np.array_equal(out.get()[0], with_zeros[np.where((ids_values[0] >= 0) & (ids_values[0] < vocab), ids_values[0], vocab)])
        row_values = rng.integers(-1, cap + 1, (1, tokens, 1))
        dest_pe, dest_row = new("int32", (tokens, 1), 0), new("int64", (tokens, 1), row_values)
        note("moe_combine_sum", tokens, dim)
        rt.moe_combine_sum("half", out.address, table.address, cap, None, dest_pe.address, dest_row.address, tokens, 1, dim)
        rt.sync()
        row = row_values[0, :, 0]
        assert np.array_equal(out.get()[0], with_zeros[np.where((row >= 0) & (row < cap), row, vocab)])


@pytest.mark.parametrize("tokens,dim,topk", [(65_600, 264, 2), (4_194_400, 3, 2)])
def test_more_sums_than_a_grid_has_rows(tokens, dim, topk):
    cap = 40
    rng = np.random.default_rng(dim)
    with runtime(1, 1 << 30) as rt, Arrays(rt) as new:
        recv_values = rng.integers(-20, 21, (cap, dim)).astype(np.float32)      # sums that fp16 holds exactly
        recv, out = new("half", (cap, dim), recv_values), new("half", (tokens, dim))
        row_values = rng.integers(-1, cap + 1, (1, tokens, topk))
        dest_pe, dest_row = new("int32", (tokens, topk), 0), new("int64", (tokens, topk), row_values)
        note("moe_combine_sum", tokens, dim, topk)
        rt.moe_combine_sum("half", out.address, recv.address, cap, None, dest_pe.address, dest_row.address, tokens, topk, dim)
        rt.sync()
        with_zeros = np.concatenate([recv_values, np.zeros((1, dim), np.float32)])
        at = np.where((row_values[0] >= 0) & (row_values[0] < cap), row_values[0], cap)
        assert np.array_equal(out.get()[0], sum(with_zeros[at[:, k]] for k in range(topk)))


@pytest.mark.parametrize("dim", [3, 10])
def test_gradients_of_more_tokens_than_a_grid_has_blocks(dim):
    tokens = (1 << 20) + 77
    rng = np.random.default_rng(dim)
    with runtime(1, 256 << 20) as rt, Arrays(rt) as new:
        recv_values = rng.integers(-8, 9, (1, tokens, dim)).astype(np.float32)
        dout_values = rng.integers(-8, 9, (1, tokens, dim)).astype(np.float32)
        row_values = rng.permutation(tokens).reshape(1, tokens, 1)
        row_values[:, ::5] = -1
        gate_values = rng.integers(1, 5, (1, tokens, 1)).astype(np.float32)
        recv, dout, gate = new("half", (tokens, dim), recv_values), new("half", (tokens, dim), dout_values), new("float", (tokens, 1), gate_values)
        dest_pe, dest_row = new("int32", (tokens, 1), 0), new("int64", (tokens, 1), row_values)
        drecv, dgate = new("half", (tokens, dim), np.float32(3)), new("float", (tokens, 1))
        note("moe_combine_grad", tokens, dim)
        rt.moe_combine_grad("half", drecv.address, dgate.address, dout.address, recv.address, tokens, gate.address, dest_pe.address,
                            dest_row.address, tokens, 1, dim)
        rt.sync()
        row, ok = row_values[0, :, 0], row_values[0, :, 0] >= 0
        want = np.full((tokens, dim), 3.0)
        want[row[ok]] = (gate_values * dout_values)[0, ok]
        assert np.array_equal(drecv.get()[0], want)
        assert np.array_equal(dgate.get()[0, :, 0], np.where(ok, (dout_values[0] * recv_values[0, np.where(ok, row, 0)]).sum(1), 0))
