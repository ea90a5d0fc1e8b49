"""Angles far past those of any position a model reaches: the header promises them to 2^50."""
from fractions import Fraction

import numpy as np
import pytest

from test_gpu_paged import Cache, served   # noqa: F401

pytestmark = pytest.mark.gpu
PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459")


def reduced(position, frequency):
    """The exact product's remainder of 2 pi, rounded to float64: 2^50 of its 2^-200 are lost."""
    angle = int(position) * Fraction(float(frequency))
    return float(angle - 2 * PI * round(angle / (2 * PI)))


@pytest.mark.parametrize("split", [False, True])
def test_angles_to_2_to_the_50(served, split):
    """Rows of (1, 0) become (cos, sin), each rounded to float32 once: half a step, and what the reduction (2^-52) and the
    series leave."""
    import torch
    positions = np.array([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 12345, 1 << 30, 1610612741, -7], np.int32)
    f = np.array([2.0 ** 19, 524287.97, 381774.87, 65537.33, 4099.7, 12.566371, 1.0, 0.0], np.float32)
    x = torch.zeros(6, 1, 16, device="cuda")
    x[..., slice(0, 8) if split else slice(0, 16, 2)] = 1
    cache = Cache([6], 4, 1, 16, "float32")
    out = served.append_rotated(x, x, cache.keys, cache.values, cache.table, cache.lengths, torch.tensor(f).cuda(),
                                torch.tensor([0, 6], dtype=torch.int32, device="cuda"), positions=torch.tensor(positions).cuda(),
                                query=x, split_half=split)[:, 0].double().cpu().numpy()
    angle = np.array([[reduced(p, w) for w in f] for p in positions])
    first, second = (slice(0, 8), slice(8, 16)) if split else (slice(0, 16, 2), slice(1, 16, 2))
    for got, want in ((out[:, first], np.cos(angle)), (out[:, second], np.sin(angle))):
        assert np.all(np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 1e-14), np.abs(got - want).max()
