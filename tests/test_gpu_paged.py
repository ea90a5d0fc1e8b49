"""The paged cache's operators against float64 (paged_reference.py), at the sizes, masks and layouts where they can
go wrong, on torch's memory and stream and on the package's own arrays."""
import numpy as np
import pytest

import paged_reference as ref
from conftest import submodule

pytestmark = pytest.mark.gpu
NAN = float("nan")


@pytest.fixture(scope="module")
def served(pkg):
    import torch
    return pkg.CUDABackend(stream=torch.cuda.current_stream().cuda_stream)


def torch_type(name):
    import torch
    return getattr(torch, name)


def wide(x):
    return x.detach().double().cpu().numpy()


class Cache:
    """Sequences of given lengths in a shuffled pool; every place that no row owns holds `garbage`."""

    def __init__(self, lengths, page, kv, dim, dtype, seed=0, garbage=NAN, extra=3, head_major=False, table_pages=None,
                 scale=1.0):
        import torch
        rng = np.random.default_rng(seed)
        need = [-(-max(n, 0) // page) for n in lengths]
        width = table_pages or max(max(need), 1)
        ids = rng.permutation(sum(need) + extra)
        self.page, self.kv, self.dim = page, kv, dim
        kind = torch_type(dtype)
        if head_major:
            pools = [torch.full((len(ids), kv, page, dim), garbage, device="cuda", dtype=kind).permute(0, 2, 1, 3)
                     for _ in range(2)]
        else:
            pools = [torch.full((len(ids), page, kv, dim), garbage, device="cuda", dtype=kind) for _ in range(2)]
        self.keys, self.values = pools
        table, at = np.full((len(lengths), width), -1, np.int32), 0
        self.rows = []
        for s, n in enumerate(lengths):
            table[s, :need[s]] = ids[at:at + need[s]]
            at += need[s]
            rows = [torch.tensor(rng.normal(size=(max(n, 0), kv, dim)) * scale).to(kind).cuda() for _ in range(2)]
            for pool, r in zip(pools, rows):
                for t in range(max(n, 0)):
                    pool[int(table[s, t // page]), t % page] = r[t]
            self.rows.append(rows)
        self.table = torch.tensor(table, device="cuda")
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.spare = [int(i) for i in ids[at:]]


def queries(batch, heads, dim, dtype, seed=1, scale=1.5):
    import torch
    return torch.tensor(np.random.default_rng(seed).normal(size=(batch, heads, dim)) * scale).to(torch_type(dtype)).cuda()


def check_paged(served, cache, q, dtype, window=None, sinks=0, weighted=False, scale=None, hidden=None, out=None):
    import torch
    batch, heads, dim = q.shape
    capacity = cache.table.shape[1] * cache.page
    weights = torch.rand(batch, cache.kv, capacity, device="cuda") if weighted else None
    before = weights.clone() if weighted else None
    got = served.paged_attention(q, cache.keys, cache.values, cache.table, cache.lengths, window=window, sinks=sinks,
                                 scale=scale, weights=weights, out=out)
    factor = dim ** -0.5 if scale is None else scale
    for s, (k, v) in enumerate(cache.rows):
        n = len(k)
        want, w, mixed, reach = ref.attend(wide(q[s:s + 1]), wide(k), wide(v), [n - 1], factor, window, sinks,
                                           hidden[s] if hidden else ())
        bound = ref.output_bound(want, mixed, reach, dim, n, dtype, False)
        assert np.all(np.abs(wide(got[s]) - want[0]) <= bound[0]), (s, np.abs(wide(got[s]) - want[0]).max())
        if weighted:
            grown = wide(weights[s]) - wide(before[s])
            spent = np.zeros((cache.kv, capacity))
            spent[:, :n] = w[0].reshape(cache.kv, heads // cache.kv, n).sum(1)
            error = 2 * ref.score_error(reach.max(), dim) + 2 * (n + heads) * 2.0 ** -24
            assert np.all(np.abs(grown - spent) <= error * spent + 2.0 ** -23 * (1 + spent))
            assert torch.equal(weights[s, :, n:], before[s, :, n:])
    return got


TYPES = ["bfloat16", "float16", "float32"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv, dim, page, lengths, window, sinks", [
    (8, 2, 32, 16, [256, 0, 1, 15, 16, 17, 33], None, 0),
    (4, 4, 64, 8, [65, 130, 7], 9, 4),
    (16, 4, 128, 32, [300, 31, 1], 64, 40),
    (6, 2, 40, 5, [23, 61], None, 0),
    (5, 1, 80, 1, [40, 3], 1, 0),
    (24, 24, 128, 64, [129, 64], 128, 1),
    (32, 1, 64, 16, [77, 50], None, 0),
    (20, 2, 96, 20, [99, 160], 30, 200),
    (40, 2, 8, 16, [50], 17, 3),
])
def test_paged_attention(served, dtype, heads, kv, dim, page, lengths, window, sinks):
    cache = Cache(lengths, page, kv, dim, dtype)
    for weighted in (False, True):
        check_paged(served, cache, queries(len(lengths), heads, dim, dtype), dtype, window, sinks, weighted)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths, window, sinks", [([2500, 3, 700], None, 0), ([2600], 2000, 11), ([900] * 3, 65, 0)])
def test_long_sequences_are_split_and_joined(served, dtype, lengths, window, sinks):
    cache = Cache(lengths, 64, 2, 64, dtype)
    check_paged(served, cache, queries(len(lengths), 8, 64, dtype), dtype, window, sinks, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv, dim, page, lengths", [(8, 2, 32, 16, [1500, 40]), (12, 4, 128, 32, [1100, 0, 690]),
                                                           (20, 2, 96, 20, [1300]), (3, 3, 40, 7, [1200, 1200])])
def test_cut_units_of_every_layout(served, dtype, heads, kv, dim, page, lengths):
    for weighted in (False, True):
        check_paged(served, Cache(lengths, page, kv, dim, dtype), queries(len(lengths), heads, dim, dtype), dtype,
                    weighted=weighted)


def test_an_infinite_value_in_a_cut_unit(served):
    import torch
    cache = Cache([3000], 16, 1, 64, "bfloat16")
    cache.values[int(cache.table[0, 40]), 3, 0, 5] = float("-inf")
    got = served.paged_attention(queries(1, 2, 64, "bfloat16"), cache.keys, cache.values, cache.table, cache.lengths)
    assert torch.isinf(got[0, :, 5]).all() and torch.isfinite(got[0, :, :5]).all() and torch.isfinite(got[0, :, 6:]).all()
    cache.values[int(cache.table[0, 40]), 3] = cache.rows[0][1][40 * 16 + 3]
    check_paged(served, cache, queries(1, 2, 64, "bfloat16"), "bfloat16")


def test_many_sequences(served):
    rng = np.random.default_rng(3)
    lengths = [int(n) for n in rng.integers(0, 40, 300)]
    check_paged(served, Cache(lengths, 16, 2, 16, "float16"), queries(300, 4, 16, "float16"), "float16", None, 0, True)


def test_four_value_heads_of_float32(served):
    check_paged(served, Cache([9, 4], 4, 2, 4, "float32"), queries(2, 4, 4, "float32"), "float32", 4, 1, True)


@pytest.mark.parametrize("dtype", TYPES)
def test_head_major_pages_and_strided_queries(served, dtype):
    import torch
    cache = Cache([100, 37], 16, 4, 64, dtype, head_major=True)
    packed = queries(2, 16 + 8, 64, dtype)
    out = torch.full((2, 40, 64), NAN, device="cuda", dtype=packed.dtype)
    got = check_paged(served, cache, packed[:, 8:], dtype, out=out[:, 8:24])
    assert got.data_ptr() == out[:, 8:].data_ptr()
    assert torch.isnan(out[:, :8]).all() and torch.isnan(out[:, 24:]).all()
    # every second sequence of a longer table and length array
    cache.table = cache.table.repeat_interleave(2, 0)[::2]
    cache.lengths = cache.lengths.repeat_interleave(2)[::2]
    check_paged(served, cache, packed[:, 8:], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [NAN, float("inf")])
def test_what_a_mask_hides_does_not_matter(served, dtype, bad):
    cache = Cache([200, 90], 16, 2, 64, dtype, garbage=bad)
    for s, n in enumerate((200, 90)):   # rows outside the window and behind the sinks
        for t in range(3, n - 20):
            for pool in (cache.keys, cache.values):
                pool[int(cache.table[s, t // 16]), t % 16] = bad
    check_paged(served, cache, queries(2, 8, 64, dtype), dtype, 20, 3, True)


@pytest.mark.parametrize("dtype", TYPES)
def test_bad_pages_hide_their_rows(served, dtype):
    import torch
    cache = Cache([100, 64, 20], 16, 2, 32, dtype)
    cache.table[0, 2], cache.table[1, 0], cache.table[2, :] = -5, 1 << 30, -1
    hidden = [set(range(32, 48)), set(range(16)), set(range(20))]
    got = check_paged(served, cache, queries(3, 4, 32, dtype), dtype, None, 0, True, hidden=hidden)
    assert not got[2].any()
    # lengths past the table and below nothing
    cache = Cache([64, 64], 16, 2, 32, dtype)
    q = queries(2, 4, 32, dtype)
    cache.lengths = torch.tensor([2 ** 31 - 1, -7], dtype=torch.int32, device="cuda")
    cache.rows[1] = [r[:0] for r in cache.rows[1]]
    assert not check_paged(served, cache, q, dtype)[1].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_scores(served, dtype):
    # one row far above the others, scores to some thousands, a negative and a zero scale
    cache = Cache([150, 70], 16, 2, 64, dtype, scale=8.0)
    q = queries(2, 8, 64, dtype, scale=8.0)
    for scale in (1.0, -0.5, 0.0):
        check_paged(served, cache, q, dtype, scale=scale, weighted=True)


def test_an_infinite_visible_value_reaches_the_output(served):
    import torch
    cache = Cache([50], 16, 1, 64, "bfloat16")
    cache.values[int(cache.table[0, 1]), 3, 0, 5] = float("inf")
    got = served.paged_attention(queries(1, 2, 64, "bfloat16"), cache.keys, cache.values, cache.table, cache.lengths)
    assert torch.isinf(got[0, :, 5]).all() and torch.isfinite(got[0, :, :5]).all()


def test_offsets_past_32_bits(served):
    import torch
    # pages 2^28 values apart: the last starts past 4 G values
    store = torch.empty((1 << 32) + (1 << 20), device="cuda", dtype=torch.bfloat16)
    pool = store.as_strided((17, 16, 2, 64), (1 << 28, 128, 64, 1))
    small = Cache([40], 16, 2, 64, "bfloat16")
    for i, page in enumerate((16, 3, 9)):
        pool[page] = small.keys[int(small.table[0, i])]
        small.table[0, i] = page
    values = torch.empty_like(store).as_strided(pool.shape, pool.stride())
    for i, page in enumerate((16, 3, 9)):
        rows = small.rows[0][1][16 * i:16 * i + 16]
        values[page, :len(rows)] = rows
    small.keys, small.values = pool, values
    q = queries(1, 4, 64, "bfloat16")
    check_paged(served, small, q, "bfloat16", weighted=True)
    new = [queries(1, 2, 64, "bfloat16", seed=s) for s in (5, 6)]
    small.lengths[0] = 7
    served.append_pages(*new, pool, values, small.table, small.lengths)
    assert torch.equal(pool[16, 6], new[0][0]) and torch.equal(values[16, 6], new[1][0])


# ---- prompts ------------------------------------------------------------------------------------------------------
def check_window(served, dtype, heads, kv, dim, new, earlier, window=None, sinks=0, garbage=NAN, scale=None, size=1.5,
                 poison=None):
    import torch
    rng = np.random.default_rng(7)
    kind = torch_type(dtype)
    keys_of = [a + b for a, b in zip(new, earlier)]
    q = torch.tensor(rng.normal(size=(sum(new) + 3, heads, dim)) * size).to(kind).cuda()
    k, v = (torch.full((sum(keys_of) + 140, kv, dim), garbage, device="cuda", dtype=kind) for _ in range(2))
    for x in (k, v):
        x[:sum(keys_of)] = torch.tensor(rng.normal(size=(sum(keys_of), kv, dim))).to(kind)
    if poison:
        poison(k, v)
    qo, ko = (torch.tensor(np.concatenate([[0], np.cumsum(x)]), dtype=torch.int32, device="cuda") for x in (new, keys_of))
    out = torch.full_like(q, 7.0)
    got = served.window_attention(q, k, v, qo, None if keys_of == new else ko, window=window, sinks=sinks, scale=scale,
                                  out=out)
    assert got is out and (got[sum(new):] == 7.0).all()
    a = b = 0
    for n, m in zip(new, keys_of):
        want, _, mixed, reach = ref.attend(wide(q[a:a + n]), wide(k[b:b + m]), wide(v[b:b + m]), range(m - n, m),
                                           dim ** -0.5 if scale is None else scale, window, sinks)
        bound = ref.output_bound(want, mixed, reach, dim, m, dtype, True)
        error = np.abs(wide(got[a:a + n]) - want)
        assert np.all(error <= bound), (n, m, np.unravel_index(np.argmax(error - bound), error.shape), error.max())
        a, b = a + n, b + m


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv, dim, new, earlier, window, sinks", [
    (8, 2, 32, [5, 1, 0, 64, 130], [0, 0, 0, 0, 0], None, 0),
    (16, 4, 64, [200, 33], [0, 0], 64, 4),
    (4, 1, 128, [150, 20], [0, 0], None, 0),
    (4, 4, 128, [140], [133], 50, 7),
    (6, 2, 40, [31, 70], [12, 0], 9, 2),
    (5, 1, 80, [40, 3, 90], [7, 300, 0], None, 0),
    (20, 2, 96, [25, 1], [260, 129], 100, 130),
    (2, 2, 16, [300], [0], 1, 0),
    (12, 1, 8, [129], [0], 129, 1),
    (48, 1, 24, [30], [5], 20, 0),
])
def test_window_attention(served, dtype, heads, kv, dim, new, earlier, window, sinks):
    check_window(served, dtype, heads, kv, dim, new, earlier, window, sinks)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_short_and_one_long_prompt(served, dtype):
    # more pieces than the GPU has SMs, several to each; and a prompt whose pieces go one to an SM
    rng = np.random.default_rng(12)
    new = [int(n) for n in rng.integers(0, 30, 50)]
    check_window(served, dtype, 4, 4, 64, new[:-1] + [0], [0] * 50, None, 0)
    check_window(served, dtype, 4, 4, 72, new, [int(n) for n in rng.integers(0, 9, 50)], 7, 2)
    check_window(served, dtype, 2, 1, 64, [1090], [0], None, 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_queries_than_keys(served, dtype):
    # the first queries stand before the first key: they see nothing and give zeros
    import torch
    q, k, v = (queries(n, h, 64, dtype, seed=n) for n, h in ((40, 4), (25, 2), (26, 2)))
    offsets = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 30, 40], [0, 10, 25])]
    got = served.window_attention(q, k, v[:25], *offsets)
    assert not got[:20].any()
    for a, b, c, d in ((20, 30, 0, 10), (30, 40, 10, 25)):
        want, _, mixed, reach = ref.attend(wide(q[a:b]), wide(k[c:d]), wide(v[c:d]), range(d - c - b + a, d - c), 0.125)
        assert np.all(np.abs(wide(got[a:b]) - want) <= ref.output_bound(want, mixed, reach, 64, 25, dtype, True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [NAN, float("inf"), float("-inf")])
def test_hidden_keys_of_a_prompt_do_not_matter(served, dtype, bad):
    import torch
    # the last rows of each sequence are bad, and some that fall out of the window again: the
    # rows that do not see them are as exact as ever (worked out another way, so not the same bits)
    q, k, v = (queries(n, h, 64, dtype, seed=n) for n, h in ((300, 4), (299, 2), (298, 2)))
    k, v = torch.cat([k, k[:1]]), torch.cat([v, v[:2]])
    offsets = torch.tensor([0, 150, 300], dtype=torch.int32, device="cuda")
    q64, k64, v64 = wide(q), wide(k), wide(v)
    for x in (k, v):
        x[141:150], x[291:300], x[2:9] = bad, bad, bad
    got = wide(served.window_attention(q, k, v, offsets, window=100, sinks=2))
    for a in (0, 150):
        want, _, mixed, reach = ref.attend(q64[a:a + 150], k64[a:a + 150], v64[a:a + 150], range(150), 0.125, 100, 2)
        bound = ref.output_bound(want, mixed, reach, 64, 150, dtype, True)
        clean = slice(109, 141) if a == 0 else slice(0, 141)
        assert np.all(np.abs(got[a:a + 150] - want)[clean] <= bound[clean])
        assert not np.isfinite(got[a + 149]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_scales_and_strides(served, dtype):
    import torch
    check_window(served, dtype, 4, 2, 64, [70], [0], scale=-0.3, size=4.0)
    check_window(served, dtype, 4, 2, 64, [70], [0], scale=0.0)
    # query, keys and values as slices of one projection's rows, and a head-major output
    rows = queries(90, 8 + 2 + 2, 64, dtype, seed=11)
    q, k, v = rows[:, :8], rows[:, 8:10], rows[:, 10:]
    out = torch.empty(8, 90, 64, device="cuda", dtype=rows.dtype).permute(1, 0, 2)
    offsets = torch.tensor([0, 90], dtype=torch.int32, device="cuda")
    a = served.window_attention(q, k, v, offsets, window=30, out=out)
    b = served.window_attention(q.contiguous(), k.contiguous(), v.contiguous(), offsets, window=30)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 104])
def test_prompts_in_other_layouts(served, dtype, dim):
    # head-major rows, keys broadcast to all heads, rows of a longer buffer read backwards in heads
    import torch
    q, k, v = (queries(130, h, dim, dtype, seed=h) for h in (4, 2, 2))
    offsets = torch.tensor([0, 60, 130], dtype=torch.int32, device="cuda")
    want = served.window_attention(q, k, v, offsets, window=50, sinks=3)
    major = [x.permute(1, 0, 2).contiguous().permute(1, 0, 2) for x in (q, k, v)]
    assert torch.equal(served.window_attention(*major, offsets, window=50, sinks=3), want)
    same = k[:, :1].expand(-1, 2, -1)
    got = served.window_attention(q, same, same, offsets, window=50, sinks=3)
    assert torch.equal(got, served.window_attention(q, same.contiguous(), same.contiguous(), offsets, window=50, sinks=3))
    row = k[7:8].expand(130, -1, -1)
    got = served.window_attention(q, row, row, offsets)
    assert torch.equal(got, served.window_attention(q, row.contiguous(), row.contiguous(), offsets))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [70, 128, 130])
def test_groups_of_many_heads(served, dtype, heads):
    check_window(served, dtype, heads, 1, 16, [9, 14], [3, 0], 5, 2)
    check_paged(served, Cache([40, 17], 8, 1, 16, dtype), queries(2, heads, 16, dtype), dtype, weighted=True)


def test_offsets_that_do_not_rise_stay_inside(served):
    import torch
    q, k = queries(20, 2, 64, "bfloat16"), queries(20, 2, 64, "bfloat16", seed=2)
    for bad in ([0, 50, 10], [-9, 5, 2 ** 31 - 1], [20, 0, 20]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        served.window_attention(q, k, k, offsets)
        served.append_pages(q, k, *(torch.zeros(2, 8, 2, 64, device="cuda", dtype=q.dtype) for _ in range(2)),
                            torch.zeros(2, 1, dtype=torch.int32, device="cuda"),
                            torch.tensor([5, 9], dtype=torch.int32, device="cuda"), offsets)
    torch.cuda.synchronize()


# ---- append -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kv, dim, page", [(2, 64, 16), (3, 40, 7), (24, 128, 32), (1, 8, 1)])
def test_append_pages(served, dtype, kv, dim, page):
    import torch
    total = [50, 0, 33, 9]
    cache = Cache(total, page, kv, dim, dtype, garbage=7.0)
    want = cache.keys.clone(), cache.values.clone()
    for s, n in enumerate(total):   # take the last rows out, as they were before the append
        for t in range(max(0, n - 12), n):
            for pool in (cache.keys, cache.values):
                pool[int(cache.table[s, t // page]), t % page] = 7.0
    counts = [min(12, n) for n in total]
    new = [torch.cat([r[i][len(r[i]) - c:] for r, c in zip(cache.rows, counts)] + [cache.rows[0][i][:2] * NAN])
           for i in range(2)]
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    served.append_pages(*new, cache.keys, cache.values, cache.table, cache.lengths, offsets)
    assert torch.equal(cache.keys, want[0]) and torch.equal(cache.values, want[1])
    # one row per sequence; the empty sequence and a bad page are passed over
    one = [queries(4, kv, dim, dtype, seed=s) for s in (1, 2)]
    cache.table[2, (33 - 1) // page] = -1
    served.append_pages(*one, cache.keys, cache.values, cache.table, cache.lengths)
    for i, (pool, was) in enumerate(zip((cache.keys, cache.values), want)):
        for s, n in ((0, 50), (3, 9)):
            was[int(cache.table[s, (n - 1) // page]), (n - 1) % page] = one[i][s]
        assert torch.equal(pool, was)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kv, dim, page", [(3, 24, 16), (1, 8, 5), (6, 64, 32)])
def test_append_many_rows(served, dtype, kv, dim, page):
    import torch
    total, counts = [410, 0, 520, 3, 90], [410, 0, 407, 3, 0]
    cache = Cache(total, page, kv, dim, dtype, garbage=7.0)
    want = cache.keys.clone(), cache.values.clone()
    for s, (n, c) in enumerate(zip(total, counts)):
        for t in range(n - c, n):
            for pool in (cache.keys, cache.values):
                pool[int(cache.table[s, t // page]), t % page] = 7.0
    new = [torch.cat([r[i][len(r[i]) - c:] for r, c in zip(cache.rows, counts)] + [cache.rows[0][i][:40] * NAN])
           for i in range(2)]
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    cache.table[2, 200 // page] = 1 << 29   # a bad page: its rows are passed over
    bad = slice(200 // page * page, 200 // page * page + page)
    served.append_pages(*new, cache.keys, cache.values, cache.table, cache.lengths, offsets)
    first = 520 - 407
    for pool, was, r in zip((cache.keys, cache.values), want, cache.rows[2]):
        hidden = [t for t in range(bad.start, bad.stop) if t >= first]
        same = (pool == was).all(-1).all(-1)
        assert int((~same).sum()) == len(hidden)          # the rows of the bad page's own place alone
        assert (pool[~same] == 7.0).all()
        assert torch.equal(was[~same], r[hidden])


# ---- eviction -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kv, dim, page, lengths, budget, sinks, recent", [
    (2, 64, 16, [200, 0, 40, 41, 90], 40, 4, 8),
    (3, 40, 7, [61, 100], 30, 0, 0),
    (1, 8, 1, [70], 9, 4, 5),
    (2, 128, 32, [300, 20], 299, 64, 20),
    (4, 16, 16, [3000], 1000, 7, 130),
    (2, 32, 8, [30, 25], 64, 3, 3),
])
def test_evict_pages(served, dtype, kv, dim, page, lengths, budget, sinks, recent):
    import torch
    cache = Cache(lengths, page, kv, dim, dtype)
    capacity = cache.table.shape[1] * page
    room = min(budget, capacity) + 5
    rng = np.random.default_rng(4)
    weights = rng.random((len(lengths), kv, capacity)).astype(np.float32)
    weights[:, 0] = np.round(weights[:, 0] * 4) / 4          # ties
    weights[0, 0, 5:9] = [np.nan, -0.0, 0.0, -np.inf]
    weights[0, 0, 11] = np.inf
    weights[0, -1, :] = 0.25
    pages = -(-room // page)
    target = torch.tensor(rng.permutation(len(lengths) * pages).reshape(len(lengths), pages).astype(np.int32)).cuda()
    pools = [torch.full((len(lengths) * pages, page, kv, dim), 7.0, device="cuda", dtype=cache.keys.dtype) for _ in range(2)]
    kept, new_lengths, new_weights = served.evict_pages(
        cache.keys, cache.values, cache.table, cache.lengths, torch.tensor(weights).cuda(), target, budget=budget,
        sinks=sinks, recent=recent, target_keys=pools[0], target_values=pools[1])
    assert kept.shape == (len(lengths), kv, budget) and new_weights.shape == (len(lengths), kv, pages * page)
    for s, n in enumerate(lengths):
        assert int(new_lengths[s]) == min(n, budget)
        for h in range(kv):
            rows = ref.evict(weights[s, h], n, budget, sinks, recent)
            assert kept[s, h].tolist() == rows + [-1] * (budget - len(rows))
            np.testing.assert_array_equal(new_weights[s, h].cpu().numpy(), np.concatenate(
                [weights[s, h, rows], np.zeros(pages * page - len(rows), np.float32)]))
            for pool, source in zip(pools, cache.rows[s]):
                moved = pool[target[s].long()].reshape(pages * page, kv, dim)[:, h]
                assert torch.equal(moved[:len(rows)], source[rows, h])
                assert (moved[len(rows):] == 7.0).all()


@pytest.mark.parametrize("rows,lengths,budget,sinks,recent,skew", [
    (40000, [40000, 28672, 28673, 4097], 20000, 4, 300, 0),   # more rows than the CTA marks at once
    (49152, [49152, 49151, 1], 49000, 0, 0, 0),               # the most that shared memory takes
    (60000, [60000, 57345, 33, 0], 31, 1, 2, 0),              # more than it takes
    (60000, [60000, 40001], 59000, 0, 1, 1),
    (5001, [5001, 3999, 2], 1000, 0, 0, 1),                   # weights on no 16-byte boundary, odd lengths
    (5001, [5001, 129], 5000, 2500, 2500, 3),
])
def test_eviction_chooses_among_many_rows(served, rows, lengths, budget, sinks, recent, skew):
    """Which rows are kept, with ties over all threads, weights alike in a whole head and strided rows of weights."""
    import torch
    heads, page = 3, 8
    pages = -(-rows // page)
    rng = np.random.default_rng(7)
    weights = (rng.random((len(lengths), heads, pages * page)) ** 4).astype(np.float32)
    weights[:, 0] = np.round(weights[:, 0] * 16) / 16
    weights[:, 1] = 0.0
    held = torch.zeros(len(lengths), heads, pages * page + skew, device="cuda")
    held[:, :, skew:] = torch.tensor(weights)
    keys = torch.zeros(pages, page, heads, 8, device="cuda", dtype=torch.bfloat16)
    room = -(-budget // page)
    target = torch.arange(len(lengths) * room, dtype=torch.int32, device="cuda").view(len(lengths), room)
    pools = [torch.empty(len(lengths) * room, page, heads, 8, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(len(lengths), 1)
    kept, new_lengths, new_weights = served.evict_pages(
        keys, keys, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), held[:, :, skew:], target, budget=budget,
        sinks=sinks, recent=recent, target_keys=pools[0], target_values=pools[1])
    kept, new_weights = kept.cpu().numpy(), new_weights.cpu().numpy()
    assert new_lengths.tolist() == [min(n, budget) for n in lengths]
    for s, n in enumerate(lengths):
        for h in range(heads):
            want = ref.evict(weights[s, h], n, budget, sinks, recent)
            assert kept[s, h].tolist() == want + [-1] * (budget - len(want))
            np.testing.assert_array_equal(new_weights[s, h, :len(want)], weights[s, h, want])
            assert not new_weights[s, h, len(want):].any()


def test_eviction_within_one_pool_and_past_bad_pages(served):
    import torch
    cache = Cache([60, 50], 8, 2, 32, "float16", extra=8)
    target = torch.tensor([cache.spare[:3], cache.spare[3:6]], dtype=torch.int32, device="cuda")
    cache.table[1, 0], target[1, 1] = -1, 10 ** 6
    before = cache.keys.clone()
    weights = torch.rand(2, 2, 64, device="cuda")
    kept, lengths, _ = served.evict_pages(cache.keys, cache.values, cache.table, cache.lengths, weights, target,
                                          budget=24, sinks=3, recent=2)
    assert lengths.tolist() == [24, 24]
    for h in range(2):
        moved = cache.keys[target[0].long()].reshape(24, 2, 32)[:, h]
        assert torch.equal(moved, cache.rows[0][0][kept[0, h].long(), h])
        moved = cache.keys[target[1, ::2].long()].reshape(16, 2, 32)[:, h]   # the bad target page is passed over
        rows = kept[1, h].long()[[*range(8), *range(16, 24)]]
        want = cache.rows[1][0][rows, h] * (rows >= 8)[:, None]              # the bad source page gives zeros
        assert torch.equal(moved, want)
    changed = [i for i in range(len(before)) if not torch.equal(before[i].nan_to_num(), cache.keys[i].nan_to_num())]
    assert set(changed) <= set(target[0].tolist()) | {int(target[1, 0]), int(target[1, 2])}


# ---- together -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
def test_serving_two_sequences(served, dtype):
    """Prompts, appends, decoded tokens with their weights, an eviction, and decoding on from what was kept."""
    import torch
    heads, kv, dim, page, prompts, steps = 8, 2, 64, 16, [70, 41], 6
    rng = np.random.default_rng(5)
    kind = torch_type(dtype)
    rows = [[torch.tensor(rng.normal(size=(n + steps + 1, h, dim))).to(kind).cuda() for h in (heads, kv, kv)]
            for n in prompts]
    pool = [torch.zeros(24, page, kv, dim, device="cuda", dtype=kind) for _ in range(2)]
    table = torch.arange(12, dtype=torch.int32, device="cuda").reshape(2, 6)
    offsets = torch.tensor([0, 70, 111], dtype=torch.int32, device="cuda")
    q, k, v = (torch.cat([r[i][:n] for r, n in zip(rows, prompts)]) for i in range(3))
    out = served.window_attention(q, k, v, offsets, window=32, sinks=4)
    lengths = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    served.append_pages(k, v, *pool, table, lengths, offsets)
    weights = torch.zeros(2, kv, 96, device="cuda")
    spent = [np.zeros((kv, n + steps)) for n in prompts]
    for step in range(steps):
        lengths += 1
        q, k, v = (torch.stack([r[i][n + step] for r, n in zip(rows, prompts)]) for i in range(3))
        served.append_pages(k, v, *pool, table, lengths)
        out = served.paged_attention(q, *pool, table, lengths, weights=weights)
        for s, n in enumerate(prompts):
            at = n + step
            want, w, mixed, reach = ref.attend(wide(rows[s][0][at:at + 1]), wide(rows[s][1][:at + 1]),
                                               wide(rows[s][2][:at + 1]), [at], dim ** -0.5)
            assert np.all(np.abs(wide(out[s]) - want[0]) <= ref.output_bound(want, mixed, reach, dim, at, dtype, False)[0])
            spent[s][:, :at + 1] += w[0].reshape(kv, heads // kv, at + 1).sum(1)
    for s, n in enumerate(prompts):
        np.testing.assert_allclose(weights[s, :, :n + steps].cpu().numpy(), spent[s], rtol=1e-4, atol=1e-6)
    target = torch.arange(12, 18, dtype=torch.int32, device="cuda").reshape(2, 3)
    kept, lengths, weights = served.evict_pages(*pool, table, lengths, weights, target, budget=40, sinks=4, recent=8)
    assert lengths.tolist() == [40, 40] and weights.shape == (2, kv, 48)
    lengths += 1
    q, k, v = (torch.stack([r[i][n + steps] for r, n in zip(rows, prompts)]) for i in range(3))
    served.append_pages(k, v, *pool, target, lengths)
    out = served.paged_attention(q, *pool, target, lengths, weights=weights)
    for s, n in enumerate(prompts):
        for h in range(kv):
            at = [*kept[s, h].tolist(), n + steps]
            group = slice(h * heads // kv, (h + 1) * heads // kv)
            want, _, mixed, reach = ref.attend(wide(q[s:s + 1, group]), wide(rows[s][1][at, h:h + 1]),
                                               wide(rows[s][2][at, h:h + 1]), [40], dim ** -0.5)
            assert np.all(np.abs(wide(out[s, group]) - want[0]) <=
                          ref.output_bound(want, mixed, reach, dim, 41, dtype, False)[0])


def test_results_repeat_bit_for_bit(served):
    import torch
    cache = Cache([1500, 700], 16, 2, 64, "bfloat16")
    q = queries(2, 8, 64, "bfloat16")
    runs = []
    for _ in range(2):
        w = torch.zeros(2, 2, cache.table.shape[1] * 16, device="cuda")
        runs.append((served.paged_attention(q, cache.keys, cache.values, cache.table, cache.lengths, weights=w), w))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])


def test_captured_calls_replay_side_by_side(pkg):
    """Two graphs of one backend, replayed on two streams at once with new inputs, and eager calls beside them."""
    import torch
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    caches = [Cache([2000, 900], 16, 2, 64, "bfloat16", seed=s) for s in range(2)]
    qs = [queries(2, 8, 64, "bfloat16", seed=s) for s in range(2)]
    target = torch.arange(8, dtype=torch.int32, device="cuda").reshape(2, 4)
    pools = [[torch.zeros(8, 16, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)] for _ in range(2)]
    capacity = caches[0].table.shape[1] * 16
    weights = [torch.zeros(2, 2, capacity, device="cuda") for _ in range(2)]
    offsets = torch.tensor([0, 900, 1000], dtype=torch.int32, device="cuda")
    prompts = [[queries(1000, h, 64, "bfloat16", seed=h + s) for h in (8, 2, 2)] for s in range(2)]
    with torch.cuda.stream(stream):
        b = pkg.CUDABackend(stream=stream.cuda_stream)
    torch.cuda.synchronize()

    def step(i):
        c = caches[i]
        out = b.paged_attention(qs[i], c.keys, c.values, c.table, c.lengths, weights=weights[i])
        kept = b.evict_pages(c.keys, c.values, c.table, c.lengths, weights[i], target, budget=64, sinks=4, recent=16,
                             target_keys=pools[i][0], target_values=pools[i][1])
        return [out, *kept, b.window_attention(*prompts[i], offsets, window=100, sinks=3)]

    graphs, results = [], []
    for i in range(2):
        with torch.cuda.stream(stream):
            step(i)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            results.append(step(i))
        graphs.append(graph)
    for i in range(2):   # new values in the captured inputs
        qs[i].copy_(queries(2, 8, 64, "bfloat16", seed=20 + i))
        weights[i].zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(stream):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    got = [[x.clone() for x in r] + [w.clone()] for r, w in zip(results, weights)]
    for i in range(2):
        weights[i].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(3):
                want = step(i)
        torch.cuda.synchronize()
        for x, y in zip(got[i], want + [weights[i]]):
            assert torch.equal(x, y)
    del graphs


def test_two_backends_on_two_streams(pkg):
    import torch
    streams = [torch.cuda.Stream() for _ in range(2)]
    backends = [pkg.CUDABackend(stream=s.cuda_stream) for s in streams]
    caches = [Cache([1900, 400, 77], 16, 2, 64, "bfloat16", seed=s) for s in range(2)]
    qs = [queries(3, 8, 64, "bfloat16", seed=s) for s in range(2)]
    outs = [[torch.empty_like(q) for _ in range(8)] for q in qs]
    torch.cuda.synchronize()
    for r in range(8):
        for i, b in enumerate(backends):
            c = caches[i]
            b.paged_attention(qs[i], c.keys, c.values, c.table, c.lengths, out=outs[i][r])
    torch.cuda.synchronize()
    for i in range(2):
        check_paged(backends[i], caches[i], qs[i], "bfloat16", out=outs[i][0].clone())
        assert all(torch.equal(x, outs[i][0]) for x in outs[i])


def test_arrays_of_the_package(backend):
    """The same calls without torch, on the backend's own stream and arrays."""
    rng = np.random.default_rng(8)
    rows = [rng.normal(size=(20, 2, 32)).astype(np.float32) for _ in range(2)]
    for dtype in TYPES:
        pools = [backend.upload_array(np.zeros((4, 8, 2, 32)), dtype) for _ in range(2)]
        k, v = (backend.upload_array(r, dtype) for r in rows)
        table, lengths, offsets = (backend.upload_array(x, "int32") for x in ([[2, 0, 3]], [20], [0, 20]))
        backend.append_pages(k, v, *pools, table, lengths, offsets)
        q = backend.upload_array(rng.normal(size=(1, 4, 32)), dtype)
        weights = backend.upload(np.zeros((1, 2, 24)))
        out = backend.paged_attention(q, *pools, table, lengths, weights=weights)
        kk, vv, qq = (backend.read_array(x).astype(np.float64) for x in (k, v, q))
        want, w, mixed, reach = ref.attend(qq, kk, vv, [19], 32 ** -0.5)
        got = backend.read_array(out).astype(np.float64)
        assert np.all(np.abs(got - want) <= ref.output_bound(want, mixed, reach, 32, 20, dtype, False))
        np.testing.assert_allclose(backend.read(weights)[0, :, :20], w[0].reshape(2, 2, 20).sum(1), rtol=1e-4)
    assert backend.read_array(backend.empty_array((0, 3), "int32")).shape == (0, 3)


def test_refusals_name_the_argument(served, pkg):
    import torch
    cache = Cache([20], 16, 2, 32, "bfloat16")
    q = queries(1, 4, 32, "bfloat16")
    with pytest.raises(pkg.CUDAError, match="one type"):
        served.paged_attention(q.half(), cache.keys, cache.values, cache.table, cache.lengths)
    with pytest.raises(ValueError, match="page_table must be on device 0, not the host"):
        served.paged_attention(q, cache.keys, cache.values, cache.table.cpu(), cache.lengths)
    with pytest.raises(ValueError, match="unsupported array type"):
        served.paged_attention(q.double(), cache.keys, cache.values, cache.table, cache.lengths)
    for bad in (0, -3, 1.5, True):
        with pytest.raises(ValueError, match="window must be"):
            served.paged_attention(q, cache.keys, cache.values, cache.table, cache.lengths, window=bad)
    with pytest.raises(ValueError, match="go together"):
        served.evict_pages(cache.keys, cache.values, cache.table, cache.lengths, torch.zeros(1, 2, 32, device="cuda"),
                           cache.table, budget=4, target_keys=cache.keys)
    with pytest.raises(pkg.CUDAError, match="room for 32 rows"):
        served.evict_pages(cache.keys, cache.values, torch.zeros(1, 4, dtype=torch.int32, device="cuda"), cache.lengths,
                           torch.zeros(1, 2, 64, device="cuda"), cache.table, budget=40)


def test_nothing_to_do(served):
    import torch
    cache = Cache([20], 16, 2, 32, "bfloat16")
    none = torch.empty(0, 4, 32, device="cuda", dtype=torch.bfloat16)
    ints = torch.empty(0, dtype=torch.int32, device="cuda")
    assert served.paged_attention(none, cache.keys, cache.values, cache.table[:0], ints).shape == (0, 4, 32)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert served.window_attention(none, none[:, :2], none[:, :2], zero).shape == (0, 4, 32)
    served.append_pages(none[:, :2], none[:, :2], cache.keys, cache.values, cache.table[:0], ints, zero)
    q = queries(2, 4, 32, "bfloat16")
    got = served.window_attention(q, none[:, :2], none[:, :2], zero.new_tensor([0, 2]), zero.new_tensor([0, 0]))
    assert not got.any()
    empty = served.paged_attention(q, cache.keys[:0], cache.values[:0], cache.table[:0].new_zeros(2, 3), zero.new_tensor([5, 9]))
    assert not empty.any()
    assert not served.paged_attention(q, cache.keys, cache.values, cache.table.new_zeros(2, 0), zero.new_tensor([5, 9])).any()
