"""Most likely tokens where the search for their bound meets an order that no logit has."""
import numpy as np
import pytest

from test_gpu_paged import served, wide   # noqa: F401
from test_gpu_scores import check

pytestmark = pytest.mark.gpu


def halved_to_minus_zero(rows, vocab, slices, b=3.5):
    """Float32 rows of -b, zeros in the first 8 of the 256 parts of each of the CTAs' `slices` (vector v of a slice belongs to
    part v % 256), and in one of those b less an ulp: the middle of the orders of -b and of the number behind that one is
    0x7fffffff, what -0 would have were both zeros not taken as equal, and 8 parts reach it."""
    x = np.full((rows, vocab), -b, np.float32)
    vectors = vocab // 4
    tops = []
    for s in range(slices):
        first, last = vectors * s // slices, vectors * (s + 1) // slices
        v = np.arange(first, last)
        at = v[(v - first) % 256 < 8]
        for j in range(4):
            x[:, at * 4 + j] = 0
        tops.append(at[len(at) // 2] * 4 + 1)
    x[:, tops] = np.nextafter(np.float32(b), np.float32(0))
    return x


@pytest.mark.parametrize("rows, vocab, slices", [
    (1600, 12000, 1),   # a warp's rows: 384 zeros and room for 256
    (300, 40000, 1),    # a CTA's: 1280, 1024
    (2, 200000, 4),     # a cluster's: 1568 a CTA
])
def test_many_zeros_behind_the_largest(served, rows, vocab, slices):
    import torch
    x = torch.tensor(halved_to_minus_zero(rows, vocab, slices)).cuda()
    for _ in range(2):
        check(served, x, 1, 4 + slices)
        x[x == 0] = -0.0
