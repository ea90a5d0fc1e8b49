"""Rotated appends, pages of 4 bits and log probabilities without a GPU: what they refuse before any device work."""
import re

import numpy as np
import pytest

import packed_reference as ref
from conftest import submodule
from test_paged_host import BF16, F16, F32, I32, Fake, append, evict, paged, refused, window

U8 = 4


def bytes_of(dim, page=16, **kw):
    shape = (10, page, 4, dim * 5 // 8)
    return Fake(shape, U8, **kw), Fake(shape, U8, pointer=1 << 24, **kw)


def rotated(**changes):
    k, v = (Fake((10, 16, 4, 64)), Fake((10, 16, 4, 64), pointer=1 << 24))
    args = dict(query=Fake((7, 8, 64)), keys=Fake((7, 4, 64)), values=Fake((7, 4, 64)), key_pages=k, value_pages=v,
                table=Fake((3, 5), I32), lengths=Fake((3,), I32), offsets=Fake((4,), I32), frequencies=Fake((32,), F32),
                positions=None, out=Fake((7, 8, 64), pointer=1 << 28), split=0)
    args.update(changes)
    values = list(args.values())
    return refused("mr_append_rotated", values[:11], *values[11:])


@pytest.mark.parametrize("changes, message", [
    (dict(), "ctx is NULL"),
    (dict(query=None, out=None, frequencies=None), "ctx is NULL"),
    (dict(positions=Fake((7,), I32), split=1), "ctx is NULL"),
    (dict(zip(("key_pages", "value_pages"), bytes_of(64))), "ctx is NULL"),
    (dict(keys=Fake((7, 4, 64), F32), values=Fake((7, 4, 64), F32), query=Fake((7, 8, 64), F32),
          out=Fake((7, 8, 64), F32, pointer=1 << 28), **dict(zip(("key_pages", "value_pages"), bytes_of(64)))), "ctx is NULL"),
    (dict(out=None), "query and out go together"),
    (dict(query=None), "query and out go together"),
    (dict(out=Fake((7, 8, 64))), "must not share memory"),
    (dict(out=Fake((7, 8, 64), F16, pointer=1 << 28)), "of one type"),
    (dict(query=Fake((6, 8, 64)), out=Fake((6, 8, 64), pointer=1 << 28)), "query must be \\[7, heads, 64\\]"),
    (dict(query=Fake((7, 8, 32)), out=Fake((7, 8, 32), pointer=1 << 28)), "query must be \\[7, heads, 64\\]"),
    (dict(frequencies=Fake((33,), F32)), "at most half of the 64 dims"),
    (dict(frequencies=Fake((32,), BF16)), "frequencies must be float32"),
    (dict(positions=Fake((6,), I32)), "positions must have 7 values"),
    (dict(positions=Fake((7,), F32)), "positions must be int32"),
    (dict(offsets=None), "one row for each of the 3 sequences"),
    (dict(values=Fake((7, 4, 64), F16)), "of one floating type"),
    (dict(keys=Fake((7, 4, 64), F16), values=Fake((7, 4, 64), F16)), "keys, values and the pages must be of one type"),
    (dict(zip(("key_pages", "value_pages"), bytes_of(128))), "\\[tokens, 4, 128\\]"),
    (dict(key_pages=bytes_of(64)[0]), "must be of one type"),
    (dict(key_pages=Fake((10, 16, 4, 64), I32), value_pages=Fake((10, 16, 4, 64), I32)), "one floating type"),
    (dict(zip(("key_pages", "value_pages"), bytes_of(64, stride=(2816, 176, 44, 1)))), "stride 2 is not a multiple of 8 bytes"),
    (dict(zip(("key_pages", "value_pages"), bytes_of(48))), "20, 40, 60 or 80 bytes"),
    (dict(zip(("key_pages", "value_pages"), (Fake((10, 16, 4, 40), U8, pointer=(1 << 20) + 4),
                                             Fake((10, 16, 4, 40), U8)))), "8-byte boundary"),
    (dict(zip(("key_pages", "value_pages"), bytes_of(64, stride=(0, 160, 40, 1)))), "must not overlap itself"),
    (dict(key_pages=None), "key_pages is missing"),
])
def test_append_rotated_refuses(changes, message):
    assert re.search(message, rotated(**changes))


def test_appends_to_pages_of_4_bits_are_checked():
    k, v = bytes_of(64)
    assert append(key_pages=k, value_pages=v) == "ctx is NULL"
    assert "of one type" in append(key_pages=k)
    assert "differ in shape" in append(key_pages=k, value_pages=Fake((9, 16, 4, 40), U8))
    assert "as the pages' heads and dim" in append(key_pages=k, value_pages=v, keys=Fake((7, 4, 32)), values=Fake((7, 4, 32)))


def read(**changes):
    k, v = bytes_of(64)
    args = dict(key_pages=k, value_pages=v, table=Fake((3, 5), I32), lengths=Fake((3,), I32), offsets=Fake((4,), I32),
                keys=Fake((90, 4, 64), pointer=1 << 27), values=Fake((90, 4, 64), pointer=1 << 28))
    args.update(changes)
    return refused("mr_read_pages", list(args.values()))


@pytest.mark.parametrize("changes, message", [
    (dict(), "ctx is NULL"),
    (dict(keys=Fake((90, 4, 64), F32, pointer=1 << 27), values=Fake((90, 4, 64), F32, pointer=1 << 28)), "ctx is NULL"),
    (dict(values=Fake((90, 4, 64), pointer=1 << 27)), "keys and values must not share memory"),
    (dict(keys=Fake((90, 4, 64))), "keys and the pages must not share memory"),
    (dict(values=Fake((90, 4, 64), pointer=1 << 24)), "values and the pages must not share memory"),
    (dict(keys=Fake((90, 4, 64), stride=(0, 64, 1))), "must not overlap itself"),
    (dict(keys=Fake((90, 4, 64), U8)), "of one floating type"),
    (dict(keys=Fake((90, 2, 64)), values=Fake((90, 2, 64), pointer=1 << 28)), "\\[tokens, 4, 64\\]"),
    (dict(offsets=None), "one row for each of the 3 sequences"),
    (dict(offsets=Fake((3,), I32)), "offsets must have 4 values"),
    (dict(key_pages=Fake((10, 16, 4, 64), F16), value_pages=Fake((10, 16, 4, 64), F16)), "of one type"),
])
def test_read_pages_refuses(changes, message):
    assert re.search(message, read(**changes))


def test_bytes_are_no_values_elsewhere():
    """uint8 arrays where values, counts or weights are asked for."""
    assert "floating type" in window(keys=Fake((90, 4, 64), U8), values=Fake((90, 4, 64), U8), query=Fake((50, 8, 64), U8),
                                     out=Fake((50, 8, 64), U8, pointer=1 << 28))
    assert "must be int32" in paged(lengths=Fake((3,), U8))
    assert "must be float32" in paged(weights=Fake((3, 4, 80), U8))
    assert "must be int32" in evict(kept=Fake((3, 4, 20), U8))


def score(**changes):
    args = dict(logits=Fake((6, 500), F32), tokens=Fake((6, 2), I32), logprobs=Fake((6, 2), F32, pointer=1 << 24),
                entropy=Fake((6,), F32), top_tokens=Fake((6, 20), I32), top_logprobs=Fake((6, 20), F32, pointer=1 << 25))
    args.update(changes)
    return refused("mr_log_probabilities", list(args.values()))


@pytest.mark.parametrize("changes, message", [
    (dict(), "ctx is NULL"),
    (dict(tokens=None, logprobs=None, entropy=None), "ctx is NULL"),
    (dict(tokens=Fake((6,), I32), logprobs=Fake((6,), F32, pointer=1 << 24), top_tokens=None, top_logprobs=None), "ctx is NULL"),
    (dict(logits=Fake((6, 500), F32, stride=(501, 1))), "ctx is NULL"),
    (dict(logits=Fake((6, 500), BF16, pointer=(1 << 20) + 2, stride=(0, 1))), "ctx is NULL"),
    (dict(logits=Fake((6, 500), I32)), "floating type"),
    (dict(logits=Fake((6, 500), U8)), "floating type"),
    (dict(logits=Fake((6, 5, 100), F32)), "must have 2 dimensions"),
    (dict(logits=Fake((6, 500), F32, stride=(1, 6))), "last dimension must be contiguous"),
    (dict(logits=Fake((6, 0), F32)), "must have a vocabulary"),
    (dict(logprobs=None), "tokens and logprobs go together"),
    (dict(top_tokens=None), "go together"),
    (dict(tokens=Fake((5, 2), I32), logprobs=Fake((5, 2), F32)), "a row for each of the 6 rows"),
    (dict(logprobs=Fake((6, 3), F32)), "differ in shape"),
    (dict(logprobs=Fake((6, 2), F16)), "logprobs must be float32"),
    (dict(logprobs=Fake((6, 2), F32)), "must not share memory"),
    (dict(tokens=Fake((6, 2), F32)), "tokens must be int32"),
    (dict(entropy=Fake((5,), F32)), "entropy must have 6 values"),
    (dict(entropy=Fake((6,), F32, stride=(0,))), "must not overlap itself"),
    (dict(top_tokens=Fake((6, 129), I32), top_logprobs=Fake((6, 129), F32)), "at most 128 tokens"),
    (dict(logits=Fake((6, 19), F32)), "at most 19 tokens"),
    (dict(top_logprobs=Fake((6, 21), F32)), "must be \\[6, 20\\]"),
    (dict(top_tokens=Fake((6, 20), F32)), "top_tokens must be int32"),
])
def test_log_probabilities_refuses(changes, message):
    assert re.search(message, score(**changes))


def test_the_format_of_4_bits():
    """A row's codes, steps and bases, and what they stand for: within half a step, and what rounding its numbers adds."""
    rng = np.random.default_rng(0)
    x = (rng.normal(size=(200, 128)) * np.exp(rng.normal(size=(200, 1)) * 3)).astype(np.float32)
    x[0] = 3.25
    x[1, :32] = 0
    rows = ref.packed(x)
    assert rows.shape == (200, 80) and rows.dtype == np.uint8
    pair = np.ascontiguousarray(rows[:, 64:]).view(np.float16).astype(np.float64).reshape(200, 4, 2)
    step, base = (np.repeat(pair[..., i], 32, axis=1) for i in range(2))
    got = ref.unpacked(rows)
    bound = step / 2 + 15 * 2.0 ** -10 * step + 2.0 ** -11 * (np.abs(base) + np.abs(got)) + 2.0 ** -24
    # a base or a step past float16 (the header: 32 values too far apart) reads as NaN, and nothing else does
    groups = x.reshape(200, 4, 32)
    spread = groups.max(-1).astype(np.float64) - groups.min(-1)
    past = np.repeat(np.abs(groups.min(-1) - 64 / 15 * spread) >= 65520 * (1 - 2.0 ** -9), 32, axis=1)
    assert np.array_equal(np.isnan(got), past) and past.any()
    assert np.all((np.abs(got - x) <= bound) | past)
    assert np.all(got[0] == 3.25) and np.all(got[1, :32] == 0)
    for bad in (np.nan, np.inf, -np.inf, 2e5):
        x[2, 40] = bad
        got = ref.unpacked(ref.packed(x[2:3]))[0]
        assert np.isnan(got[32:64]).all() and np.isfinite(got[:32]).all() and np.isfinite(got[64:]).all()


def test_arrays_of_bytes():
    arrays = submodule("arrays")
    assert arrays.host_type("uint8") == np.uint8
    assert arrays.TYPES["uint8"] == U8

    class Owner:
        shape, dtype = (2,), "float32"

        def new_empty(self, shape, dtype=None):
            return shape, dtype

    assert arrays.empty_like(Owner(), (3, 0), "int32") == ((3, 0), "int32")
    assert arrays.empty_like(Owner(), (3,), "float32") == ((3,), None)
    import torch
    made = arrays.empty_like(torch.zeros(2, dtype=torch.bfloat16), (4, 1), "float32")
    assert made.dtype == torch.float32 and made.shape == (4, 1)


def test_attention_and_eviction_of_4_bits_are_checked():
    k, v = bytes_of(64)
    both = dict(key_pages=k, value_pages=v)
    assert paged(**both) == "ctx is NULL"
    assert paged(query=Fake((3, 8, 64), F32), out=Fake((3, 8, 64), F32, pointer=1 << 28), **both) == "ctx is NULL"
    assert "of one floating type" in paged(out=Fake((3, 8, 64), F32, pointer=1 << 28), **both)
    assert "of one floating type" in paged(query=Fake((3, 8, 64), I32), out=Fake((3, 8, 64), I32, pointer=1 << 28), **both)
    assert "of one type" in paged(key_pages=k)
    assert "32 values a head, the pages 64" in paged(query=Fake((3, 8, 32)), out=Fake((3, 8, 32), pointer=1 << 28), **both)
    far = bytes_of(64, stride=(1 << 32, 160, 40, 1))
    assert "stride 0 passes 4 GB" in paged(key_pages=far[0], value_pages=far[1])
    assert evict(target_keys=k, target_values=v, **both) == "ctx is NULL"
    assert "target_keys and target_values must be of one type" in evict(**both)
