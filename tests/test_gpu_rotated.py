"""Appends with a rotation, into pages of the rows' type and of 4 bits, and rows read back, against packed_reference.py."""
import numpy as np
import pytest

import packed_reference as ref
from conftest import submodule
from test_gpu_paged import NAN, TYPES, Cache, queries, served, torch_type, wide   # noqa: F401

pytestmark = pytest.mark.gpu
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def frequencies(n, theta=1e4):
    import torch
    return torch.tensor(theta ** (-np.arange(n) / max(n, 1)), dtype=torch.float32, device="cuda")


def offsets_of(counts):
    import torch
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")


def turn_bound(want, size, dtype):
    """Two products, a sum and the sines, each rounded to float32 (2^-24 of the parts); then the type's rounding."""
    tiny = 2.0 ** -25 if dtype == "float16" else 0.0
    return HALF_STEP[dtype] * np.abs(want) + (1 + HALF_STEP[dtype]) * 3 * 2.0 ** -24 * size + tiny + 1e-30


class Pages4:
    """Pages of 4 bits for sequences of given lengths; bytes that no row owns hold `garbage`."""

    def __init__(self, lengths, page, kv, dim, seed=0, garbage=255, extra=3, head_major=True, table_pages=None):
        import torch
        rng = np.random.default_rng(seed)
        need = [-(-max(n, 0) // page) for n in lengths]
        ids = rng.permutation(sum(need) + extra)
        self.page, self.kv, self.dim = page, kv, dim
        shape = (len(ids), kv, page, dim * 5 // 8) if head_major else (len(ids), page, kv, dim * 5 // 8)
        self.keys, self.values = (torch.full(shape, garbage, dtype=torch.uint8, device="cuda") for _ in range(2))
        if head_major:
            self.keys, self.values = (x.permute(0, 2, 1, 3) for x in (self.keys, self.values))
        table, at = np.full((len(lengths), table_pages or max(max(need), 1)), -1, np.int32), 0
        for s in range(len(lengths)):
            table[s, :need[s]] = ids[at:at + need[s]]
            at += need[s]
        self.spare = [int(i) for i in ids[at:]]
        self.table = torch.tensor(table, device="cuda")
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def rows(self, s, rows):
        """The bytes of a sequence's rows, on the host: keys, values [rows, kv, bytes]."""
        at = [(int(self.table[s, t // self.page]), t % self.page) for t in rows]
        return [np.stack([x[p, r].cpu().numpy() for p, r in at]) if at else np.zeros((0, self.kv, self.dim * 5 // 8), np.uint8)
                for x in (self.keys, self.values)]


CASES = [   # heads, kv, dim, page, lengths, new rows, n, theta
    (8, 2, 32, 16, [50, 3, 0, 17], [12, 3, 0, 1], 16, 1e4),
    (16, 4, 64, 8, [65, 130], [65, 7], 32, 1e4),
    (4, 4, 128, 64, [300, 1], [200, 1], 64, 5e5),
    (6, 2, 40, 5, [23, 61], [23, 30], 10, 1e4),
    (5, 1, 96, 7, [40, 33], [9, 33], 48, 1e4),
    (3, 3, 24, 16, [29], [29], 5, 1e4),      # an odd number of pairs, a part of the dims
    (2, 1, 8, 1, [9], [8], 3, 10.0),
    (12, 1, 128, 16, [70], [64], 32, 1e4),   # half of the dims
    (4, 2, 16, 4, [21], [21], 0, 1e4),       # nothing turns
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("heads, kv, dim, page, lengths, new, n, theta", CASES)
def test_append_rotated(served, dtype, split, heads, kv, dim, page, lengths, new, n, theta):
    import torch
    cache = Cache(lengths, page, kv, dim, dtype, garbage=7.0)
    total = sum(new)
    q, k, v = (queries(total + 2, h, dim, dtype, seed=i) for i, h in enumerate((heads, kv, kv)))
    out = torch.full_like(q, 7.0)
    before = cache.keys.clone(), cache.values.clone()
    got = served.append_rotated(k, v, cache.keys, cache.values, cache.table, cache.lengths, frequencies(n, theta),
                                offsets_of(new), query=q, out=out, split_half=split)
    assert got is out and (out[total:] == 7.0).all()
    rows = np.concatenate([np.arange(a - c, a) for a, c in zip(lengths, new)])
    f = frequencies(n, theta).cpu().numpy()
    want, size = ref.turned64(wide(q[:total]), rows, f, split)
    assert np.all(np.abs(wide(out[:total]) - want) <= turn_bound(want, size, dtype))
    want, size = ref.turned64(wide(k[:total]), rows, f, split)
    at = 0
    for s, (a, c) in enumerate(zip(lengths, new)):
        for t in range(a - c, a):
            place = int(cache.table[s, t // page]), t % page
            assert np.all(np.abs(wide(cache.keys[place]) - want[at]) <= turn_bound(want[at], size[at], dtype))
            assert torch.equal(cache.values[place], v[at])
            before[0][place], before[1][place] = cache.keys[place], cache.values[place]
            at += 1
    assert torch.equal(before[0], cache.keys) and torch.equal(before[1], cache.values)   # and nothing else was written


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("split", [False, True])
def test_given_and_far_positions(served, dtype, split):
    """Positions of both signs to 2^31: the angle is the exact product, whatever its size."""
    import torch
    cache = Cache([6, 2], 4, 2, 64, dtype)
    positions = np.array([0, -3, 131071, 10 ** 6 + 7, 2 ** 31 - 1, -2 ** 31, 5, 77777777], np.int32)
    f = np.concatenate([[1.0, 0.7390851], 1e4 ** (-np.arange(30) / 30)]).astype(np.float32)
    q, k = queries(8, 3, 64, dtype), queries(8, 2, 64, dtype, seed=2)
    out = served.append_rotated(k, k, cache.keys, cache.values, cache.table, cache.lengths,
                                torch.tensor(f).cuda(), offsets_of([6, 2]), positions=torch.tensor(positions).cuda(),
                                query=q, split_half=split)
    # 2^31 x 0.739 has more bits than 64-bit floating point: angles reduced in 80 bits
    exact = positions.astype(np.longdouble)[:, None] * f.astype(np.longdouble)
    pi = np.longdouble("3.14159265358979323846264338327950288")
    angle = (exact - 2 * pi * np.rint(exact / (2 * pi))).astype(np.float64)
    x = wide(q)
    n = 32
    first, second = (slice(0, n), slice(n, 64)) if split else (slice(0, 64, 2), slice(1, 64, 2))
    z = (x[..., first] + 1j * x[..., second]) * np.exp(1j * angle)[:, None]
    size = (np.abs(x[..., first]) + np.abs(x[..., second])) * (1 + 2.0 ** -8)   # 80 bits leave 2^31 x 2^-63: below 2^-24 / 100
    for part, at in ((z.real, first), (z.imag, second)):
        assert np.all(np.abs(wide(out)[..., at] - part) <= turn_bound(part, size, dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_one_row_a_sequence_and_layouts(served, dtype):
    """A decode step without offsets: rows of one projection, a head-major pool, strided counts, no query."""
    import torch
    cache = Cache([100, 0, 37, 16], 16, 4, 64, dtype, head_major=True)
    rows = queries(4, 8 + 4 + 4, 64, dtype)
    out = torch.full((4, 20, 64), 7.0, device="cuda", dtype=rows.dtype)
    lengths = cache.lengths.repeat_interleave(2)[::2]
    f = frequencies(32).repeat_interleave(3)[::3]
    served.append_rotated(rows[:, 8:12], rows[:, 12:], cache.keys, cache.values, cache.table, lengths, f,
                          query=rows[:, :8], out=out[:, 4:12])
    assert (out[:, :4] == 7.0).all() and (out[:, 12:] == 7.0).all()
    position = np.array([99, -1, 36, 15])
    want, size = ref.turned64(wide(rows[:, :12]), position, f.cpu().numpy(), False)
    bound = turn_bound(want, size, dtype)
    assert np.all(np.abs(wide(out[:, 4:12]) - want[:, :8]) <= bound[:, :8])   # the empty sequence's query too
    for s in (0, 2, 3):
        place = int(cache.table[s, position[s] // 16]), position[s] % 16
        assert np.all(np.abs(wide(cache.keys[place]) - want[s, 8:]) <= bound[s, 8:])
        assert torch.equal(cache.values[place], rows[s, 12:])
    assert served.append_rotated(rows[:, 8:12], rows[:, 12:], cache.keys, cache.values, cache.table, lengths, f) is None


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_have_no_place(served, dtype):
    """Bad pages, more new rows than the sequence is long, lengths past the table, offsets that do not rise."""
    import torch
    cache = Cache([40, 5, 64], 16, 2, 32, dtype, garbage=7.0)
    cache.table[0, 1] = 1 << 29
    before = cache.keys.clone(), cache.values.clone()
    k, v, q = (queries(60, h, 32, dtype, seed=h) for h in (2, 2, 4))
    cache.lengths[2] = 70   # six rows past the table
    new = [20, 9, 10]
    out = served.append_rotated(k, v, cache.keys, cache.values, cache.table, cache.lengths, frequencies(16),
                                offsets_of(new), query=q)
    position = np.concatenate([np.arange(20, 40), np.arange(-4, 5), np.arange(60, 70)])
    f = frequencies(16).cpu().numpy()
    want, size = ref.turned64(wide(q[:39]), position, f, False)
    assert np.all(np.abs(wide(out[:39]) - want) <= turn_bound(want, size, dtype))
    for i, (s, t) in enumerate([(s, t) for s, rows in ((0, range(20, 40)), (1, range(-4, 5)), (2, range(60, 70))) for t in rows]):
        if t < 0 or t >= 64 or (s, t // 16) == (0, 1):
            continue
        place = int(cache.table[s, t // 16]), t % 16
        assert torch.equal(cache.values[place], v[i])
        before[0][place], before[1][place] = cache.keys[place], v[i]
    assert torch.equal(before[0], cache.keys) and torch.equal(before[1], cache.values)
    for bad in ([0, 50, 10, 60], [-9, 5, 2 ** 31 - 1, 3], [60, 0, 60, 0]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        served.append_rotated(k, v, cache.keys, cache.values, cache.table, cache.lengths, frequencies(16), offsets, query=q)
        served.read_pages(cache.keys, cache.values, cache.table, cache.lengths, offsets, torch.empty_like(k), torch.empty_like(v))
    torch.cuda.synchronize()


# ---- 4 bits -------------------------------------------------------------------------------------------------------
def values_of(rng, tokens, kv, dim, dtype):
    """Rows of many sizes, with groups that are constant, zero, not finite or past float16."""
    import torch
    x = rng.normal(size=(tokens, kv, dim)) * np.exp(rng.normal(size=(tokens, kv, 1)))
    x[0, 0, :32] = 0.75
    x[1, 0, :32] = 0.0
    x[2, 0, 5], x[3, 0, 6], x[4, 0, 7] = NAN, np.inf, -np.inf
    x[5, 0, 3] = 6e4          # with its neighbours past what float16's base can be
    x[6, 0, :32] *= 1e-6      # steps among float16's smallest numbers
    return torch.tensor(x).to(torch_type(dtype)).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("head_major", [True, False])
@pytest.mark.parametrize("kv, dim, page, lengths, new", [(2, 32, 16, [50, 3, 0, 17], [12, 3, 0, 1]),
                                                         (4, 64, 8, [65, 130], [65, 7]), (1, 96, 7, [40, 33], [9, 33]),
                                                         (3, 128, 64, [300, 1], [200, 1]), (8, 128, 1, [9], [9])])
def test_append_to_4_bits(served, dtype, head_major, kv, dim, page, lengths, new):
    """Bytes as the format's definition gives them, bit for bit, and no others touched."""
    import torch
    rng = np.random.default_rng(4)
    pages = Pages4(lengths, page, kv, dim, head_major=head_major)
    total = sum(new)
    k, v = (values_of(rng, total + 2, kv, dim, dtype) for _ in range(2))
    want = [x.clone() for x in (pages.keys, pages.values)]
    served.append_pages(k, v, pages.keys, pages.values, pages.table, pages.lengths, offsets_of(new))
    at = 0
    for s, (a, c) in enumerate(zip(lengths, new)):
        for t in range(a - c, a):
            place = int(pages.table[s, t // page]), t % page
            for pool, x in zip(want, (k, v)):
                pool[place] = torch.tensor(ref.packed(x[at].float().cpu().numpy())).cuda()
            at += 1
    assert torch.equal(want[0], pages.keys) and torch.equal(want[1], pages.values)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("heads, kv, dim, page, lengths, new, n, theta", [c for c in CASES if c[2] in (32, 64, 96, 128)])
def test_append_rotated_to_4_bits(served, dtype, split, heads, kv, dim, page, lengths, new, n, theta):
    import torch
    pages = Pages4(lengths, page, kv, dim)
    total = sum(new)
    q, k, v = (queries(total, h, dim, dtype, seed=i) for i, h in enumerate((heads, kv, kv)))
    f = frequencies(n, theta)
    out = served.append_rotated(k, v, pages.keys, pages.values, pages.table, pages.lengths, f, offsets_of(new), query=q,
                                split_half=split)
    rows = np.concatenate([np.arange(a - c, a) for a, c in zip(lengths, new)])
    want, size = ref.turned64(wide(q), rows, f.cpu().numpy(), split)
    assert np.all(np.abs(wide(out) - want) <= turn_bound(want, size, dtype))
    turned = ref.turned32(k.float().cpu().numpy(), rows, f.cpu().numpy(), split)
    at = 0
    for s, (a, c) in enumerate(zip(lengths, new)):
        got_k, got_v = pages.rows(s, range(a - c, a))
        np.testing.assert_array_equal(got_k, ref.packed(turned[at:at + c]))
        np.testing.assert_array_equal(got_v, ref.packed(v[at:at + c].float().cpu().numpy()))
        at += c
    assert torch.equal(out, served.append_rotated(k, v, pages.keys, pages.values, pages.table, pages.lengths, f,
                                                  offsets_of(new), query=q, split_half=split))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kv, dim, page, lengths, last", [(2, 32, 16, [50, 3, 0, 17], [50, 2, 0, 17]),
                                                          (4, 64, 8, [65, 130], [60, 130]), (1, 96, 7, [40, 33], [9, 33]),
                                                          (3, 128, 64, [300, 1], [300, 1]), (2, 128, 1, [2500], [2500])])
def test_read_pages(served, dtype, kv, dim, page, lengths, last):
    import torch
    rng = np.random.default_rng(6)
    pages = Pages4(lengths, page, kv, dim)
    total = sum(lengths)
    k, v = (values_of(rng, max(total, 7), kv, dim, dtype)[:total] for _ in range(2))
    served.append_pages(k, v, pages.keys, pages.values, pages.table, pages.lengths, offsets_of(lengths))
    if last[0] > page:
        pages.table[0, 0] = -1
    got = served.read_pages(pages.keys, pages.values, pages.table, pages.lengths, offsets_of(last),
                            *(torch.full((sum(last) + 2, kv, dim), 7.0, device="cuda", dtype=k.dtype) for _ in range(2)))
    for x, source in zip(got, (k, v)):
        assert (x[sum(last):] == 7.0).all()
        at = begin = 0
        for s, (n, m) in enumerate(zip(lengths, last)):
            want = torch.tensor(ref.unpacked(ref.packed(source[begin + n - m:begin + n].float().cpu().numpy()))).to(k.dtype)
            if s == 0 and last[0] > page:
                want[:max(0, page - (n - m))] = 0.0   # the bad page's rows
            assert torch.equal(x[at:at + m].cpu().nan_to_num(5e4), want.nan_to_num(5e4))
            at, begin = at + m, begin + n


@pytest.mark.parametrize("dtype", TYPES)
def test_reading_pages_of_the_rows_type(served, dtype):
    import torch
    cache = Cache([50, 0, 9, 33], 8, 3, 40, dtype)
    k, v = (torch.full((60, 3, 40), 7.0, device="cuda", dtype=cache.keys.dtype) for _ in range(2))
    served.read_pages(cache.keys, cache.values, cache.table, cache.lengths, offsets_of([20, 0, 9, 10]), k, v)
    for i, x in enumerate((k, v)):
        assert torch.equal(x[:39], torch.cat([cache.rows[0][i][30:], cache.rows[2][i], cache.rows[3][i][23:]]))
        assert (x[39:] == 7.0).all()
    # the newest rows; more rows than there are: zeros before the first
    served.read_pages(cache.keys, cache.values, cache.table, cache.lengths, None, k[:4], v[:4])
    assert torch.equal(k[0], cache.rows[0][0][49]) and not k[1].any() and torch.equal(v[3], cache.rows[3][1][32])
    served.read_pages(cache.keys, cache.values, cache.table, cache.lengths, offsets_of([0, 2, 11, 0]), k, v)
    assert not k[:4].any() and torch.equal(k[4:13], cache.rows[2][0])


def test_offsets_past_32_bits(served):
    """Pages of 4 bits 2^31 bytes apart, rows of keys and values 2^31 bytes apart."""
    import torch
    store = [torch.empty((1 << 32) + (1 << 20), device="cuda", dtype=torch.uint8) for _ in range(2)]
    pools = [x.as_strided((3, 4, 2, 80), (1 << 31, 160, 80, 1)) for x in store]
    wide_rows = torch.empty((1 << 31) + (1 << 12), device="cuda", dtype=torch.bfloat16)
    k = wide_rows.as_strided((3, 2, 128), (1 << 30, 128, 1))
    v = queries(3, 2, 128, "bfloat16")
    k.copy_(queries(3, 2, 128, "bfloat16", seed=3))
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([3], dtype=torch.int32, device="cuda")
    served.append_pages(k, v, *pools, table, lengths, offsets_of([3]))
    for pool, x in zip(pools, (k, v)):
        assert np.array_equal(pool[2, :3].cpu().numpy(), ref.packed(x.float().cpu().numpy()))
    back = torch.zeros_like(v), torch.empty_like(v)
    served.read_pages(*pools, table, lengths, offsets_of([3]), *back)
    assert np.array_equal(wide(back[0]), wide(torch.tensor(ref.unpacked(ref.packed(k.float().cpu().numpy()))).bfloat16()))


def test_nothing_to_append_or_read(served):
    import torch
    pages = Pages4([20], 16, 2, 32)
    none = torch.empty(0, 2, 32, device="cuda", dtype=torch.bfloat16)
    ints = torch.empty(0, dtype=torch.int32, device="cuda")
    served.append_pages(none, none, pages.keys, pages.values, pages.table[:0], ints)
    served.append_rotated(none, none, pages.keys, pages.values, pages.table[:0], ints, frequencies(16), query=none)
    q = queries(1, 2, 32, "bfloat16")
    empty = pages.keys[:0]
    out = served.append_rotated(q, q, empty, empty, pages.table, pages.lengths, frequencies(16), query=q)   # no page at all
    want, size = ref.turned64(wide(q), np.array([19]), frequencies(16).cpu().numpy(), False)
    assert np.all(np.abs(wide(out) - want) <= turn_bound(want, size, "bfloat16"))
    k, v = torch.ones_like(q), torch.ones_like(q)
    served.read_pages(empty, empty, pages.table, pages.lengths, None, k, v)
    assert not k.any() and not v.any()


def test_captured_appends(pkg):
    import torch
    stream = torch.cuda.Stream()
    b = pkg.CUDABackend(stream=stream.cuda_stream)
    pages = Pages4([40, 9], 16, 2, 64)
    k, v, q = (queries(2, h, 64, "bfloat16", seed=h) for h in (2, 2, 4))
    f = frequencies(32)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = b.append_rotated(k, v, pages.keys, pages.values, pages.table, pages.lengths, f, query=q)
    k.copy_(queries(2, 2, 64, "bfloat16", seed=9))
    pages.lengths -= 3
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    turned = ref.turned32(k.float().cpu().numpy(), np.array([36, 5]), f.cpu().numpy(), False)
    for s, t in enumerate((36, 5)):
        np.testing.assert_array_equal(pages.rows(s, [t])[0], ref.packed(turned[s:s + 1]))
    want, size = ref.turned64(wide(q), np.array([36, 5]), f.cpu().numpy(), False)
    assert np.all(np.abs(wide(out) - want) <= turn_bound(want, size, "bfloat16"))


def test_bytes_of_the_package(backend):
    """Without torch: pages of 4 bits as the backend's own arrays."""
    rng = np.random.default_rng(8)
    k, v = (rng.normal(size=(20, 2, 64)).astype(np.float32) for _ in range(2))
    pools = [backend.upload_array(np.zeros((4, 8, 2, 40)), "uint8") for _ in range(2)]
    table, lengths, offsets = (backend.upload_array(x, "int32") for x in ([[2, 0, 3]], [20], [0, 20]))
    rows = [backend.upload(x) for x in (k, v)]
    backend.append_pages(*rows, *pools, table, lengths, offsets)
    held = backend.read_array(pools[0])
    assert held.dtype == np.uint8
    np.testing.assert_array_equal(held[2], ref.packed(k[:8]))
    back = [backend.empty_array((20, 2, 64), "float16") for _ in range(2)]
    backend.read_pages(*pools, table, lengths, offsets, *back)
    np.testing.assert_array_equal(backend.read_array(back[1]), ref.unpacked(ref.packed(v)).astype(np.float16))


def test_wrong_arguments_are_named(served, pkg):
    import torch
    pages = Pages4([20], 16, 2, 32)
    q = queries(1, 2, 32, "bfloat16")
    with pytest.raises(pkg.CUDAError, match="at most half"):
        served.append_rotated(q, q, pages.keys, pages.values, pages.table, pages.lengths, frequencies(17))
    with pytest.raises(ValueError, match="query must be a device array"):
        served.append_rotated(q, q, pages.keys, pages.values, pages.table, pages.lengths, frequencies(16), query=3)
    with pytest.raises(ValueError, match="frequencies must be on device 0, not the host"):
        served.append_rotated(q, q, pages.keys, pages.values, pages.table, pages.lengths, frequencies(16).cpu())
    with pytest.raises(pkg.CUDAError, match="must not share memory"):
        served.read_pages(pages.keys, pages.values, pages.table, pages.lengths, None, q, q)
    with pytest.raises(pkg.CUDAError, match="one type"):
        served.append_pages(q, q, pages.keys, torch.zeros_like(pages.keys, dtype=torch.bfloat16), pages.table, pages.lengths)
