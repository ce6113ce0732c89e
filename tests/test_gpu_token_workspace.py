"""One workspace, of the largest batch, for smaller batches that are cut into more blocks or parts than it."""
import numpy as np
import pytest

import token_reference as R
from gpu_util import note, runtime
from token_util import Arrays, close, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("largest,batches,experts", [(8192, (1024, 1000, 65, 2048), 64), (4096, (512, 256, 300), 300)])
def test_router(largest, batches, experts):
    npes, topk = 8, 4
    rng = np.random.default_rng(largest)
    with runtime(npes, 128 << 20) as rt, Arrays(rt) as new:
        ws = new.workspace("moe_route", largest, experts)
        for tokens in batches:
            # (a few rows over and over: the reference goes through them one by one)
            some = rounded(rng.standard_normal((npes, 61, experts)), "bfloat16")
            turn = np.arange(tokens) % 61
            logits = new("bfloat16", (tokens, experts), some[:, turn])
            expert, gate, counts = new("int32", (tokens, topk)), new("float", (tokens, topk)), new("int64", (experts,))
            loss, balance = new("float", (1,)), new("float", (experts,))
            note("moe_route", largest, tokens, experts)
            rt.moe_route("bfloat16", expert.address, gate.address, counts.address, ws.address, logits.address, tokens, experts, topk,
                         loss.address, balance.address)
            rt.sync()
            want = R.route(some, topk, True, 1.0)[0][:, turn]
            want_counts = np.stack([np.bincount(want[pe].reshape(-1), minlength=experts) for pe in range(npes)])
            assert np.array_equal(expert.get(), want) and np.array_equal(counts.get(), want_counts)
            b = experts * want_counts.sum(0) / (npes * npes * float(tokens) * tokens * topk)
            close(balance.get(), np.broadcast_to(b, (npes, experts)), 1.01 * R.STEP * b, "balance")
            ws.get()                                    # (looks at the guard bytes)
            for a in (logits, expert, gate, counts, loss, balance):
                a.get()


def test_tables():
    npes, topk, experts, largest = 8, 8, 32, 16384
    rng = np.random.default_rng(3)
    with runtime(npes, 128 << 20) as rt, Arrays(rt) as new:
        ws = new.workspace("moe_place", largest, topk, experts)
        for tokens in (16129, 16383, 8192):
            first = rng.integers(0, experts // topk, (npes, tokens, 1))
            e = (first * topk + np.arange(topk)).astype(np.int32)
            counts_values = np.stack([np.bincount(e[pe].reshape(-1), minlength=experts) for pe in range(npes)])
            expert, counts = new("int32", (tokens, topk), e), new("int64", (experts,), counts_values)
            dest_pe, dest_row = new("int32", (tokens, topk)), new("int64", (tokens, topk))
            expected, expert_row = new("int64", (npes,)), new("int64", (experts // npes + 1,))
            note("moe_place", largest, tokens)
            rt.moe_place(dest_pe.address, dest_row.address, expected.address, expert_row.address, ws.address, expert.address,
                         counts.address, tokens, topk, experts, 1 << 40)
            rt.sync()
            # rows in the order (expert, source PE, token): on each PE's own, counted from its first expert's
            order = np.argsort(e.reshape(-1), kind="stable")
            row = np.empty(order.size, np.int64)
            row[order] = np.arange(order.size)
            owner = e.reshape(-1) // (experts // npes)
            row -= np.searchsorted(np.sort(owner), owner)
            assert np.array_equal(dest_pe.get().reshape(-1), owner) and np.array_equal(dest_row.get().reshape(-1), row)
            ws.get()
            for a in (expert, counts, dest_pe, dest_row, expected, expert_row):
                a.get()


def test_gradient_of_the_table():
    npes, vocab, dim, largest = 8, 1003, 7168, 1207
    rng = np.random.default_rng(4)
    rows = -(-vocab // npes)
    with runtime(npes, 128 << 20) as rt, Arrays(rt) as new:
        ws = new.workspace("embedding_grad", largest, vocab, dim)
        for tokens in (329, 600, 64):
            ids_values = rng.integers(0, vocab, (npes, tokens))
            ids_values[:, ::3] = 7                      # (a sum that goes through many parts)
            dout_values = rng.integers(-8, 9, (npes, tokens, dim)).astype(np.float32)
            ids, dout, dtable = new("int64", (tokens,), ids_values), new("bfloat16", (tokens, dim), dout_values), new("bfloat16", (rows, dim))
            note("embedding_grad", largest, tokens)
            rt.embedding_grad("bfloat16", dtable.address, dout.address, ids.address, ws.address, tokens, vocab, dim, 1.0)
            rt.sync()
            want, _, _ = R.embedding_grad(np.zeros((npes, rows, dim)), dout_values, ids_values, vocab, 1.0)
            assert np.array_equal(dtable.get().reshape(-1, dim)[:vocab], rounded(want, "bfloat16").reshape(-1, dim)[:vocab])
            ws.get()
            for a in (ids, dout, dtable):
                a.get()
