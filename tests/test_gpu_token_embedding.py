"""Embedding lookup from a table cut over the PEs, and its gradient, against 64 bits."""
import numpy as np
import pytest

import token_reference as R
from gpu_util import note, runtime
from nvshmem_amd import hip
from token_util import Arrays, EPS, TINY, close, rounded

pytestmark = pytest.mark.gpu


def _ids(rng, npes, tokens, vocab, how):
    if how == "padding":
        ids = rng.integers(-2, vocab + 2, (npes, tokens))
        ids[rng.random((npes, tokens)) < 0.2] = -(1 << 62)
        ids[rng.random((npes, tokens)) < 0.1] = (1 << 32) + 1      # (row 1 if the upper half were cut off)
        return ids
    if how == "one":
        return np.full((npes, tokens), vocab - 1)
    if how == "none":
        return np.full((npes, tokens), -1)
    if how == "zipf":
        return np.minimum(np.exp(rng.random((npes, tokens)) * np.log(vocab)).astype(np.int64) - 1, vocab - 1)
    return rng.integers(0, vocab, (npes, tokens))


SIZES = [  # npes, tokens, vocab, dim, shift of the rows' buffers in elements
    (4, 5, 37, 8, 0), (8, 64, 1000, 512, 0), (8, 1, 9, 1, 0), (3, 33, 100, 1029, 1), (4, 130, 50, 63, 3),
    (16, 70, 17, 520, 0), (2, 700, 3, 136, 2), (8, 9, 3, 2049, 0), (1, 40, 64, 100, 5)]


@pytest.mark.parametrize("npes,tokens,vocab,dim,shift", SIZES)
@pytest.mark.parametrize("kind", ["float", "half", "bfloat16"])
def test_lookup(kind, npes, tokens, vocab, dim, shift):
    rng = np.random.default_rng(dim)
    rows = -(-vocab // npes)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        table_values = rounded(rng.standard_normal((npes, rows, dim)), kind)
        table = new(kind, (rows, dim), table_values, shift)
        for how in ("any", "padding", "one", "none"):
            ids_values = _ids(rng, npes, tokens, vocab, how)
            ids = new("int64", (tokens,), ids_values)
            for scale in (1.0, -2.5, 0.0):
                out = new(kind, (tokens, dim), shift=shift)
                note("embedding", kind, npes, tokens, vocab, dim, how, scale)
                rt.embedding(kind, out.address, table.address, ids.address, tokens, vocab, dim, scale)
                rt.sync()
                ok = (ids_values >= 0) & (ids_values < vocab)
                found = table_values.reshape(-1, dim)[np.where(ok, ids_values, 0)]
                # one product in fp32 and one rounding: the same bits
                want = rounded(np.where(ok[..., None], found * np.float32(scale), np.float32(0)), kind)
                got = out.get()
                assert np.array_equal(got, want) and not np.signbit(got[~ok]).any()


@pytest.mark.parametrize("npes,tokens,vocab,dim,shift", [  # wavefronts with four tokens, and with three or four chunks a lane
    (8, 700, 999, 509, 1), (8, 513, 999, 252, 0), (3, 1367, 100, 511, 0), (8, 4097, 77, 72, 2), (16, 4099, 1000, 20, 0),
    (1, 4096, 5, 256, 0), (4, 77, 130, 769, 1), (4, 77, 130, 1021, 0), (4, 77, 130, 1531, 3), (2, 90, 7, 1544, 0), (2, 90, 7, 2045, 1)])
@pytest.mark.parametrize("kind", ["float", "half", "bfloat16"])
def test_lookup_of_many_and_of_wider_rows(kind, npes, tokens, vocab, dim, shift):
    rng = np.random.default_rng(dim)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        table_values = rounded(rng.standard_normal((npes, -(-vocab // npes), dim)), kind)
        table = new(kind, table_values.shape[1:], table_values, shift)
        ids_values = _ids(rng, npes, tokens, vocab, "padding")
        ids, out = new("int64", (tokens,), ids_values), new(kind, (tokens, dim), shift=shift)
        note("embedding", kind, npes, tokens, vocab, dim)
        rt.embedding(kind, out.address, table.address, ids.address, tokens, vocab, dim, 0.5)
        rt.sync()
        ok = (ids_values >= 0) & (ids_values < vocab)
        found = table_values.reshape(-1, dim)[np.where(ok, ids_values, 0)]
        # half of a value is exact but for fp16's subnormals, which round once
        assert np.array_equal(out.get(), rounded(np.where(ok[..., None], found * np.float32(0.5), np.float32(0)), kind))


@pytest.mark.parametrize("how", ["any", "padding", "one", "none", "zipf"])
@pytest.mark.parametrize("npes,tokens,vocab,dim,shift", SIZES)
@pytest.mark.parametrize("kind", ["float", "half", "bfloat16"])
def test_gradient(kind, npes, tokens, vocab, dim, shift, how):
    rng = np.random.default_rng(dim + 1)
    rows, scale = -(-vocab // npes), 1.5
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        dout_values = rounded(rng.standard_normal((npes, tokens, dim)), kind)
        before = rounded(rng.standard_normal((npes, rows, dim)), kind)
        ids_values = _ids(rng, npes, tokens, vocab, how)
        dout, ids = new(kind, (tokens, dim), dout_values, shift), new("int64", (tokens,), ids_values)
        dtable, ws = new(kind, (rows, dim), before, shift), new.workspace("embedding_grad", tokens, vocab, dim)
        note("embedding_grad", kind, npes, tokens, vocab, dim, how)
        rt.embedding_grad(kind, dtable.address, dout.address, ids.address, ws.address, tokens, vocab, dim, scale)
        rt.sync()
        got = dtable.get()
        want, size, n = R.embedding_grad(before, dout_values, ids_values, vocab, scale)
        # n terms added one to the other in fp32, in whatever order: n - 1 roundings of at most the sum of magnitudes; one
        # for the product with the scale, one of the result to its type
        close(got, want, (n[..., None] + 1) * R.STEP * size * 1.01 + EPS[kind] / 2 * np.abs(want) * 1.01 + TINY[kind], "dtable")
        first = got.copy()
        dtable.put(before)
        rt.embedding_grad(kind, dtable.address, dout.address, ids.address, ws.address, tokens, vocab, dim, scale)
        rt.sync()
        assert np.array_equal(dtable.get(), first), "the same inputs gave other bits"
        ws.get()


@pytest.mark.parametrize("npes,tokens,vocab", [(8, 1024, 300), (8, 1025, 70000), (4, 8191, 200000), (8, 4500, 70001), (2, 40000, 5),
                                               (16, 3001, 1 << 20)])
def test_gradient_of_many_tokens(npes, tokens, vocab):
    """Counts around what one way of sorting takes, ids of one digit and of several, and a row that most tokens name."""
    rng = np.random.default_rng(tokens)
    rows, dim = -(-vocab // npes), 3
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        ids_values = _ids(rng, npes, tokens, vocab, "zipf")
        ids_values[rng.random((npes, tokens)) < 0.3] = vocab // 2
        ids_values[rng.random((npes, tokens)) < 0.1] = -1
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


def test_infinities_and_nan_stay_in_their_rows():
    with runtime(2, 16 << 20) as rt, Arrays(rt) as new:
        dim, tokens, vocab = 70, 40, 10
        ids_values = np.arange(2 * tokens).reshape(2, tokens) % 7
        ids_values[1, -3:] = -1
        dout_values = np.ones((2, tokens, dim), np.float32)
        dout_values[0, 3], dout_values[1, 0, 5], dout_values[1, -3:] = np.nan, np.inf, np.nan   # ids 3 and 5, and padding
        dout, ids = new("float", (tokens, dim), dout_values), new("int64", (tokens,), ids_values)
        dtable, ws = new("float", (5, dim), np.float32(1)), new.workspace("embedding_grad", tokens, vocab, dim)
        rt.embedding_grad("float", dtable.address, dout.address, ids.address, ws.address, tokens, vocab, dim, 1.0)
        rt.sync()
        want, _, _ = R.embedding_grad(np.ones((2, 5, dim)), dout_values, ids_values, vocab, 1.0)
        assert np.array_equal(dtable.get(), want, equal_nan=True) and np.isnan(want).any() and np.isinf(want).any()


def test_gradient_is_the_lookups():
    """<dout, lookup(table + h d)> by differences, in fp32 with values that it holds exactly."""
    rng = np.random.default_rng(5)
    npes, tokens, vocab, dim, scale = 4, 50, 23, 20, 2.0
    rows = -(-vocab // npes)
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        table_values = rng.integers(-50, 50, (npes, rows, dim)).astype(np.float32)
        step = rng.integers(-9, 9, (npes, rows, dim)).astype(np.float32)
        dout_values = rng.integers(-9, 9, (npes, tokens, dim)).astype(np.float32)
        ids_values = _ids(rng, npes, tokens, vocab, "padding")
        ids, dout = new("int64", (tokens,), ids_values), new("float", (tokens, dim), dout_values)
        table, out = new("float", (rows, dim)), new("float", (tokens, dim))
        value = []
        for sign in (1, -1):
            table.put(table_values + sign * step)
            rt.embedding("float", out.address, table.address, ids.address, tokens, vocab, dim, scale)
            rt.sync()
            value.append((out.get().astype(np.float64) * dout_values).sum())
        dtable, ws = new("float", (rows, dim), np.float32(0)), new.workspace("embedding_grad", tokens, vocab, dim)
        rt.embedding_grad("float", dtable.address, dout.address, ids.address, ws.address, tokens, vocab, dim, scale)
        rt.sync()
        assert (value[0] - value[1]) / 2 == (dtable.get().astype(np.float64) * step).sum()


def test_no_tokens():
    with runtime(4, 16 << 20) as rt, Arrays(rt) as new:
        dtable = new("half", (3, 33), np.float32(4))
        rt.embedding("half", None, dtable.address, None, 0, 12, 33)
        rt.embedding_grad("half", dtable.address, None, None, None, 0, 11, 33)
        rt.sync()
        want = np.zeros((4, 3, 33))
        want[3, 2] = 4      # (row 11 is behind the vocabulary)
        assert np.array_equal(dtable.get(), want)


def test_on_a_stream_and_in_a_graph():
    """Replays with other ids in the same buffers, eager calls in between."""
    rng = np.random.default_rng(9)
    npes, tokens, vocab, dim = 8, 300, 5000, 70
    rows = -(-vocab // npes)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        table_values = rng.integers(-50, 50, (npes, rows, dim)).astype(np.float32)
        table, out = new("float", (rows, dim), table_values), new("float", (tokens, dim))
        ids, dtable = new("int64", (tokens,)), new("float", (rows, dim))
        ws = new.workspace("embedding_grad", tokens, vocab, dim)
        stream = hip.Stream()

        def calls(s):
            rt.embedding("float", out.address, table.address, ids.address, tokens, vocab, dim, 1.0, stream=s)
            rt.embedding_grad("float", dtable.address, out.address, ids.address, ws.address, tokens, vocab, dim, 1.0, stream=s)

        with hip.Graph(stream) as graph:
            calls(stream)
        for turn in range(4):
            ids_values = _ids(rng, npes, tokens, vocab, "zipf" if turn % 2 else "padding")
            ids.put(ids_values)
            ok = (ids_values >= 0) & (ids_values < vocab)
            want_out = np.where(ok[..., None], table_values.reshape(-1, dim)[np.where(ok, ids_values, 0)], 0)
            want, _, _ = R.embedding_grad(np.zeros((npes, rows, dim)), want_out, ids_values, vocab, 1.0)
            for run in (graph.launch, lambda: calls(stream)):
                out.put(np.float32(0))
                dtable.put(np.float32(0))
                hip.synchronize()
                run()
                stream.synchronize()
                assert np.array_equal(out.get(), want_out)
                assert np.array_equal(dtable.get(), want)
        graph.destroy()
        stream.destroy()


def test_rows_beyond_4_gib():
    """A row whose offset in its PE's copy passes 32 bits."""
    vocab, dim, tokens = 2 * 300_000, 8192, 3
    with runtime(2, 10 << 30) as rt:
        table, out = rt.malloc(300_000 * dim * 2), rt.malloc(tokens * dim * 2)
        ids, ws = rt.malloc(tokens * 8), rt.malloc(rt.workspace_bytes("embedding_grad", tokens, vocab, dim))
        rt.fill(table, 0, 300_000 * dim * 2)
        last = np.full(dim, 0x3C00, np.uint16)       # 1.0
        for pe in range(2):
            rt.upload(table, pe, last, (300_000 - 1 - pe) * dim * 2)
            rt.upload(ids, pe, np.array([299_999, 599_998, -1], np.int64))
        rt.embedding("half", out, table, ids, tokens, vocab, dim, 2.0)
        rt.sync()
        got = rt.download_all(out, (tokens, dim), np.float16)
        assert (got[:, :2] == 2).all() and (got[:, 2] == 0).all()
        rt.embedding_grad("half", table, out, ids, ws, tokens, vocab, dim, 1.0)
        rt.sync()
        for pe in range(2):
            got = rt.download(table, pe, (4, dim), np.float16, (300_000 - 4) * dim * 2)
            want = np.zeros((4, 1), np.float16)
            want[3 - pe] = 4
            assert (got == want).all()
        for p in (table, out, ids, ws):
            rt.free(p)
