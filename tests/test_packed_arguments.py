"""Arguments of the rotated appends and log probabilities that are told from good ones before any device work."""
import re

import numpy as np
import pytest

from test_packed_host import U8, Fake, bytes_of, rotated


@pytest.mark.parametrize("changes, message", [
    (dict(keys=Fake((7, 4, 64), pointer=1 << 28)), "keys and out must not share memory"),
    (dict(values=Fake((7, 4, 64), pointer=1 << 28)), "values and out must not share memory"),
    # heads of their own for each query: the key buffer has the query's shape
    (dict(query=Fake((7, 4, 64)), out=Fake((7, 4, 64), pointer=1 << 26), keys=Fake((7, 4, 64), pointer=1 << 26)),
     "keys and out must not share memory"),
    (dict(key_pages=Fake((10, 16, 4, 64), pointer=1 << 28)), "the pages and out must not share memory"),
    (dict(value_pages=Fake((10, 16, 4, 64), pointer=1 << 28)), "the pages and out must not share memory"),
    (dict(key_pages=Fake((10, 16, 4, 40), U8, pointer=1 << 28), value_pages=bytes_of(64)[1]),
     "the pages and out must not share memory"),
    # inputs may share theirs: keys that are values, and both a part of what the queries are
    (dict(keys=Fake((7, 4, 64)), values=Fake((7, 4, 64)), query=Fake((7, 8, 64))), "ctx is NULL"),
    (dict(query=None, out=None, keys=Fake((7, 4, 64), pointer=1 << 28)), "ctx is NULL"),
])
def test_turned_queries_have_memory_of_their_own(changes, message):
    assert re.search(message, rotated(**changes))


class Logits:
    """An array whose owner makes others like it; no memory is behind it."""

    shape, dtype = (2, 5), "float32"

    def new_empty(self, shape, dtype=None):
        return self


@pytest.mark.parametrize("arguments, message", [
    (dict(logits=np.zeros((2, 5), np.float32)), "logits must be a device array, not ndarray"),
    (dict(logits=[[1.0, 2.0]]), "logits must be an array"),
    (dict(logits=Logits(), tokens=[1, 2]), "tokens must be a device array, not list"),
    (dict(logits=Logits(), tokens=[1, 2], logprobs=Logits()), "must be a device array"),
    (dict(logits=Logits(), top=2, top_tokens=[1]), "top_tokens must be a device array, not list"),
    (dict(logits=Logits(), top=2, top_tokens=Logits()), "top_tokens must be \\[2, 2\\]"),
])
def test_what_is_no_device_array_is_named(pkg, arguments, message):
    backend = object.__new__(pkg.CUDABackend)   # of no context: nothing gets that far
    backend._where = 0, 0
    with pytest.raises(ValueError, match=message):
        backend.log_probabilities(**arguments)
