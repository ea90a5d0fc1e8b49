"""Arguments of the rotated appends and log probabilities that are told from good ones before any device work."""
import re

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
