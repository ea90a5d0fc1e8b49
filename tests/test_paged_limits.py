"""Sizes past what the paged cache's kernels count in 32 bits are refused, on the host."""
import pytest

from test_paged_host import Fake, paged


@pytest.mark.parametrize("heads, dim, message", [((1 << 25) - 4, 64, "ctx is NULL"), (1 << 25, 64, "too many heads"),
                                                 ((1 << 24) - 4, 128, "ctx is NULL"), (1 << 24, 128, "too many heads")])
def test_heads_and_values_of_one_query(heads, dim, message):
    pools = [Fake((10, 16, 4, dim), pointer=1 << n) for n in (20, 24)]
    changes = dict(query=Fake((1, heads, dim)), out=Fake((1, heads, dim), pointer=1 << 40), key_pages=pools[0],
                   value_pages=pools[1], lengths=Fake((1,), 3), table=Fake((1, 5), 3))
    assert message in paged(**changes)
