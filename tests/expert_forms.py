"""Calls of the experts' block that together reach every form of its kernels (tile sizes, types, ways of rows into LDS, of 4 bits): sizes
alone decide, and capacity stands for rows there, so that experts of every number of rows meet every form."""
import numpy as np

NPES, MINE = 2, 64
ROWS = [0, 1, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129]
MORE = [128, 200, 255, 257, 32, 2]

KINDS = ["bfloat16", "half", "float"]
# (name, capacity in rows of an expert, dim, hidden)
CALLS = [("12 rows", 12, 264, 136), ("32 rows", 32, 264, 136), ("100 rows", 100, 264, 136), ("449 rows", 449, 264, 136),
         ("12 odd rows", 12, 263, 137), ("32 odd rows", 32, 263, 137), ("100 odd rows", 100, 263, 137)]
# (name, capacity in rows of an expert, dim, hidden, group): of 4 bits, eight experts a PE
FOUR_BIT_CALLS = [("%d rows by %d%s" % (rows, group, odd and " odd"), rows, dim, hidden, group)
                  for odd, dim, hidden in (("", 288, 160), ("odd", 263, 137)) for group in (32, 64, 128)
                  for rows in ((100, 300) if not odd else (100,))]
FOUR_BIT_MINE = 8


def table(rng, npes, mine, cap, sizes):
    """expert_row of every PE: experts of `sizes` rows, as many as there is room for, and experts without; in an order of their own."""
    rows = np.zeros((npes, mine + 1), np.int64)
    for pe in range(npes):
        n = np.zeros(mine, np.int64)
        fit = np.cumsum(sizes) <= cap
        n[:len(sizes)] = np.where(fit, sizes, 0)[:mine]
        rows[pe, 1:] = np.cumsum(rng.permutation(n))
    return rows


FOUR_BIT_ROWS = [1, 129, 33, 65, 64, 17, 0, 200]
