"""Results of one-token attention over pages of 4 bits in bfloat16: rounded once, from sums that are far closer."""
import numpy as np
import pytest

import packed_reference as packed
import paged_reference as ref
from test_gpu_packed import Cache4, score_error
from test_gpu_paged import queries, served, wide   # noqa: F401

pytestmark = pytest.mark.gpu


def bfloat16(x):
    """Float64 rounded to bfloat16, ties to even; by its bits, 45 of the fraction's 52 going."""
    bits = np.ascontiguousarray(x, np.float64).view(np.uint64)
    low = (bits >> np.uint64(45)) & np.uint64(1)
    return ((bits + np.uint64((1 << 44) - 1) + low) >> np.uint64(45) << np.uint64(45)).view(np.float64)


def test_the_rounding_on_the_host():
    import torch
    x = np.random.default_rng(0).normal(size=1000).astype(np.float32)
    x[:3] = 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -1 - 2.0 ** -8
    assert np.array_equal(bfloat16(x.astype(np.float64)), torch.tensor(x).to(torch.bfloat16).double().numpy())


@pytest.mark.parametrize("heads, kv, dim, lengths, window", [
    (8, 2, 64, [2, 3, 5, 9, 40], None),       # four heads a group
    (16, 2, 32, [2, 3, 5, 9, 40], None),      # eight
    (6, 6, 128, [2, 7, 30], None),            # one
    (24, 2, 96, [2, 7, 30], None),            # twelve: two blocks
    (8, 2, 64, [1500, 40, 2100], 7),          # a window
    (8, 1, 32, [1100, 40, 60, 3], None),      # sequences cut and joined, and whole ones beside them
])
def test_bfloat16_results_are_rounded_once(served, heads, kv, dim, lengths, window):
    """Each result lies between the roundings of the exact one less and plus what float32 work may be off by: scores (in a
    weight twice, of numerator and sum), weights' 2^-22, and 2^-40 of the largest, the rows' 32-bit additions twice, and
    a division.  A small scale keeps the scores' part small; then the two roundings are mostly one number, and a weight of
    one float16 part alone (2^-11) puts 3 to 7 of 100 results of few rows outside (float64 simulation)."""
    cache = Cache4(lengths, 16, kv, dim, seed=heads)
    q = queries(len(lengths), heads, dim, "bfloat16")
    scale = 0.05 * dim ** -0.5
    got = wide(served.paged_attention(q, cache.keys, cache.values, cache.table, cache.lengths, window=window, scale=scale))
    for s, (k, v) in enumerate(cache.stored):
        x = wide(q[s:s + 1])
        want, _, mixed, reach = ref.attend(x, k, v, [len(k) - 1], scale, window)
        rows = min(window or len(k), len(k))
        error = 2 * (ref.score_error(reach, dim) + score_error(x, k, reach, scale, "bfloat16"))
        error = (error + 2.0 ** -22 + 2 * (rows + 8) * 2.0 ** -24) * mixed + 2.0 ** -23 * np.abs(want)
        error += 2.0 ** -40 * rows * np.abs(v).max()
        low, high = bfloat16(want - error)[0], bfloat16(want + error)[0]
        assert rows > 100 or (low == high).mean() > 0.75
        bad = (got[s] < low) | (got[s] > high)
        assert not bad.any(), (s, int(bad.sum()), bad.size)
