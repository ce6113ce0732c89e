"""Dropout on rows of tokens against its definition in whole numbers."""
import numpy as np
import pytest

from dropout_reference import kept
from gpu_util import note, runtime
from nvshmem_amd import hip
from token_util import EPS, TINY, Arrays, close, rounded

pytestmark = pytest.mark.gpu

KINDS = ["bfloat16", "half", "float"]


SEED = [0x0123456789abcdef, 0xfedcba9876543210]


def signed(seed):
    return np.array(seed, np.uint64).view(np.int64)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,dim", [(1, 1), (1, 7), (3, 8), (5, 1029), (33, 264), (64, 7168)])
@pytest.mark.parametrize("p,residual,shift", [(0.0, True, 0), (0.1, True, 1), (0.5, False, 0), (0.999, False, 3)])
def test_values(kind, tokens, dim, p, residual, shift):
    npes = 3
    rng = np.random.default_rng(tokens * dim)
    limit = int(np.rint(np.float32(p).astype(np.float64) * 65536))
    with runtime(npes, 32 << 20) as rt, Arrays(rt) as new:
        x_values = rounded(rng.standard_normal((npes, tokens, dim)), kind)
        keep = np.stack([kept(tokens * dim, pe, SEED, limit).reshape(tokens, dim) for pe in range(npes)])
        x_values[~keep] = rng.choice([np.nan, np.inf, -np.inf, 1.0], (~keep).sum())      # nothing of what is dropped comes through
        r_values = rounded(rng.standard_normal((npes, tokens, dim)), kind)
        x, seed = new(kind, (tokens, dim), x_values, shift), new("int64", (2,), signed(SEED))
        r = new(kind, (tokens, dim), r_values, shift) if residual else None
        out = new(kind, (tokens, dim), None, shift)
        note("dropout", kind, tokens, dim, p, residual, shift)
        rt.dropout(kind, out.address, x.address, seed.address, tokens, dim, p, residual=r.address if r else None)
        rt.sync()
        scaled = np.where(keep, np.where(keep, x_values, 0).astype(np.float64) * (65536.0 / (65536 - limit)), 0)
        want = scaled + (r_values if residual else 0)
        # the scale, its product and the sum are rounded to fp32, the result to the type: by half a step of its value, or, among
        # halves under 2^-14, whose step is 2^-24 whatever the value, by 2^-25 (TINY)
        close(out.get(), want, 3 * 2.0 ** -24 * (np.abs(scaled) + np.abs(want)) + EPS[kind] / 2 * 1.01 * np.abs(want) + TINY[kind] + 2.0 ** -126)
        if residual:                                                                    # in place
            rt.dropout(kind, r.address, x.address, seed.address, tokens, dim, p, residual=r.address)
            rt.sync()
            assert np.array_equal(r.get(), out.get())
        else:
            rt.dropout(kind, x.address, x.address, seed.address, tokens, dim, p)
            rt.sync()
            assert np.array_equal(x.get(), out.get())


def test_gradient_has_the_same_mask_and_another_step_another():
    npes, tokens, dim, p = 2, 64, 512, 0.25
    with runtime(npes, 32 << 20) as rt, Arrays(rt) as new:
        ones = new("float", (tokens, dim), np.float32(1))
        out, dx, seed = new("float", (tokens, dim)), new("float", (tokens, dim)), new("int64", (2,), signed(SEED))
        note("dropout masks")
        rt.dropout("float", out.address, ones.address, seed.address, tokens, dim, p)
        rt.dropout("float", dx.address, ones.address, seed.address, tokens, dim, p)
        rt.sync()
        first = out.get() != 0
        assert np.array_equal(out.get(), dx.get())
        seed.put(signed([SEED[0], SEED[1] + 1]))
        rt.dropout("float", out.address, ones.address, seed.address, tokens, dim, p)
        rt.sync()
        second = out.get() != 0
        n = first[0].size
        for mask in (first[0], first[1], second[0], second[1]):
            assert abs(mask.mean() - 0.75) < 6 * np.sqrt(0.25 * 0.75 / n)
        # any two agree where two independent ones do
        for a, b in ((first[0], first[1]), (first[0], second[0]), (second[0], second[1])):
            assert abs((a == b).mean() - 0.625) < 6 * np.sqrt(0.375 * 0.625 / n)


def test_replayed_graph_reads_the_seed_of_its_time():
    npes, tokens, dim, p = 2, 40, 264, 0.3
    limit = int(np.rint(np.float32(p).astype(np.float64) * 65536))
    with runtime(npes, 32 << 20) as rt, Arrays(rt) as new:
        ones, out, seed = new("float", (tokens, dim), np.float32(1)), new("float", (tokens, dim)), new("int64", (2,), signed(SEED))
        stream = hip.Stream()
        note("dropout graph")
        with hip.Graph(stream) as graph:
            rt.dropout("float", out.address, ones.address, seed.address, tokens, dim, p, stream=stream)
        for step in range(3):
            seed.put(signed([SEED[0], step]))
            graph.launch()
            stream.synchronize()
            for pe in range(npes):
                assert np.array_equal(out.get()[pe].reshape(-1) != 0, kept(tokens * dim, pe, [SEED[0], step], limit))
        graph.destroy()
        stream.destroy()
