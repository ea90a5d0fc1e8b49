"""One-token attention over pages of 4 bits, and evictions of them, against float64 over what their bytes stand for."""
import numpy as np
import pytest

import packed_reference as packed
import paged_reference as ref
from test_gpu_paged import NAN, TYPES, queries, served, torch_type, wide   # noqa: F401
from test_gpu_rotated import Pages4, frequencies, offsets_of

pytestmark = pytest.mark.gpu


class Cache4(Pages4):
    """Rows of random values, quantised on the host; bytes that no row owns are 255: NaN steps and bases."""

    def __init__(self, lengths, page, kv, dim, seed=0, scale=1.0, **kw):
        import torch
        super().__init__(lengths, page, kv, dim, seed=seed, **kw)
        rng = np.random.default_rng(seed + 100)
        self.stored = []
        for s, n in enumerate(lengths):
            rows = [packed.packed((rng.normal(size=(max(n, 0), kv, dim)) * scale).astype(np.float32)) for _ in range(2)]
            t = np.arange(max(n, 0))
            ids = self.table[s].cpu().numpy()[t // page]
            for pool, x in zip((self.keys, self.values), rows):
                if len(t):
                    pool[torch.tensor(ids).long().cuda(), torch.tensor(t % page).cuda()] = torch.tensor(x).cuda()
            self.stored.append([packed.unpacked(x) for x in rows])


def score_error(q, k, reach, factor, dtype):
    """What a score is off by, beside 32-bit sums: queries in float16 parts, which lose 2^-39 of a head's largest value, or of
    float32 2^-22 of a value."""
    top = np.abs(k).max() if len(k) else 0.0
    largest = np.abs(q).max(-1)[..., None] * top * abs(factor)
    return 2.0 ** -39 * q.shape[-1] * largest + (2.0 ** -21 * reach if dtype == "float32" else 0.0)


def operand_error(q, k, v, mixed, reach, factor, dtype):
    """Scores' errors in a weight twice (numerator and sum); weights in two float16 parts (2^-22, and 2^-40 of the largest),
    for bfloat16 in one."""
    weights = 2.0 ** -11 if dtype == "bfloat16" else 2.0 ** -22
    return (2 * score_error(q, k, reach, factor, dtype) + weights) * mixed + 2.0 ** -40 * len(v) * (np.abs(v).max() if len(v) else 0)


def check(served, cache, q, dtype, window=None, sinks=0, weighted=False, scale=None, hidden=None, out=None):
    import torch
    batch, heads, dim = q.shape
    capacity = cache.table.shape[1] * cache.page
    weights = torch.rand(batch, cache.kv, capacity, device="cuda") if weighted else None
    before = weights.clone() if weighted else None
    got = served.paged_attention(q, cache.keys, cache.values, cache.table, cache.lengths, window=window, sinks=sinks,
                                 scale=scale, weights=weights, out=out)
    factor = dim ** -0.5 if scale is None else scale
    for s, (k, v) in enumerate(cache.stored):
        n = len(k)
        want, w, mixed, reach = ref.attend(wide(q[s:s + 1]), k, v, [n - 1], factor, window, sinks, hidden[s] if hidden else ())
        bound = ref.output_bound(want, mixed, reach, dim, n, dtype, False)
        bound = bound + operand_error(wide(q[s:s + 1]), k, v, mixed, reach, factor, dtype)
        assert np.all(np.abs(wide(got[s]) - want[0]) <= bound[0]), (s, np.abs(wide(got[s]) - want[0]).max(), bound.max())
        if weighted:
            grown = wide(weights[s]) - wide(before[s])
            spent = np.zeros((cache.kv, capacity))
            spent[:, :n] = w[0].reshape(cache.kv, heads // cache.kv, n).sum(1)
            error = 2 * (ref.score_error(reach.max(), dim) + score_error(wide(q[s:s + 1]), k, reach, factor, dtype).max())
            error += 2 * (n + heads) * 2.0 ** -24
            assert np.all(np.abs(grown - spent) <= error * spent + 2.0 ** -23 * (1 + spent))
            assert torch.equal(weights[s, :, n:], before[s, :, n:])
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv, dim, page, lengths, window, sinks", [
    (8, 2, 32, 16, [256, 0, 1, 31, 32, 33, 65], None, 0),
    (4, 4, 64, 8, [65, 130, 7], 9, 4),
    (16, 4, 128, 32, [300, 31, 1], 64, 40),
    (5, 1, 96, 1, [40, 3], 1, 0),
    (12, 12, 128, 64, [129, 64], 128, 1),
    (32, 1, 64, 16, [77, 50], None, 0),
    (20, 2, 96, 20, [99, 160], 30, 200),
    (9, 3, 32, 5, [23, 61], None, 0),
    (40, 2, 32, 16, [50], 17, 3),
])
def test_attention_over_4_bits(served, dtype, heads, kv, dim, page, lengths, window, sinks):
    for head_major in (True, False):
        cache = Cache4(lengths, page, kv, dim, head_major=head_major)
        check(served, cache, queries(len(lengths), heads, dim, dtype), dtype, window, sinks, head_major)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv, dim, page, lengths, window, sinks", [
    (8, 2, 64, 64, [5000, 3, 700], None, 0), (8, 2, 128, 64, [5200], 4000, 11), (4, 2, 32, 16, [1500] * 3, None, 0),
    (20, 2, 96, 20, [2600, 1100], None, 0), (12, 4, 128, 32, [2100, 0, 1390], None, 0), (3, 3, 64, 7, [1200, 2200], 1500, 33)])
def test_long_sequences_are_split_and_joined(served, dtype, heads, kv, dim, page, lengths, window, sinks):
    cache = Cache4(lengths, page, kv, dim)
    for weighted in (False, True):
        check(served, cache, queries(len(lengths), heads, dim, dtype), dtype, window, sinks, weighted)


def test_many_sequences(served):
    rng = np.random.default_rng(3)
    lengths = [int(n) for n in rng.integers(0, 70, 300)]
    check(served, Cache4(lengths, 16, 2, 64), queries(300, 4, 64, "float16"), "float16", None, 0, True)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_queries_and_outputs(served, dtype):
    import torch
    cache = Cache4([100, 37], 16, 4, 64)
    rows = queries(2, 16 + 8, 64, dtype)
    out = torch.full((2, 40, 64), 7.0, device="cuda", dtype=rows.dtype)
    got = check(served, cache, rows[:, 8:], dtype, out=out[:, 8:24])
    assert got.data_ptr() == out[:, 8:].data_ptr()
    assert (out[:, :8] == 7.0).all() and (out[:, 24:] == 7.0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_what_a_mask_hides_does_not_matter(served, dtype):
    import torch
    cache = Cache4([200, 90], 16, 2, 64)
    for s, n in enumerate((200, 90)):   # rows outside the window and behind the sinks: bytes of NaN
        t = torch.arange(3, n - 20, device="cuda")
        for pool in (cache.keys, cache.values):
            pool[cache.table[s, t // 16].long(), t % 16] = 255
    check(served, cache, queries(2, 8, 64, dtype), dtype, 20, 3, True)
    out = served.paged_attention(queries(2, 8, 64, dtype), cache.keys, cache.values, cache.table, cache.lengths)
    assert torch.isnan(out).all()   # visible, they reach everything


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite_reach_their_dims(served, dtype):
    """A group of NaN in a visible value row: its 32 dims alone, of all the heads that share it."""
    import torch
    for n in (50, 3000):
        cache = Cache4([n], 16, 2, 96)
        row = packed.packed(np.concatenate([np.ones(40), [np.inf], np.ones(55)]).astype(np.float32)[None])[0]
        cache.values[int(cache.table[0, 1]), 3, 1] = torch.tensor(row).cuda()
        got = served.paged_attention(queries(1, 4, 96, dtype), cache.keys, cache.values, cache.table, cache.lengths)
        assert torch.isfinite(got[0, :2]).all() and torch.isnan(got[0, 2:, 32:64]).all()
        assert torch.isfinite(got[0, 2:, :32]).all() and torch.isfinite(got[0, 2:, 64:]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_bad_pages_hide_their_rows(served, dtype):
    import torch
    cache = Cache4([100, 64, 20], 16, 2, 32)
    cache.table[0, 2], cache.table[1, 0], cache.table[2, :] = -5, 1 << 30, -1
    hidden = [set(range(32, 48)), set(range(16)), set(range(20))]
    got = check(served, cache, queries(3, 4, 32, dtype), dtype, None, 0, True, hidden=hidden)
    assert not got[2].any()
    cache = Cache4([64, 64], 16, 2, 128)
    q = queries(2, 4, 128, dtype)
    cache.lengths = torch.tensor([2 ** 31 - 1, -7], dtype=torch.int32, device="cuda")
    cache.stored[1] = [r[:0] for r in cache.stored[1]]
    assert not check(served, cache, q, dtype)[1].any()
    assert not served.paged_attention(q, cache.keys[:0], cache.values[:0], cache.table, cache.lengths).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_scores_and_queries(served, dtype):
    """One row far above the others, negative and zero scales, queries whose heads are of very different sizes."""
    cache = Cache4([150, 70], 16, 2, 64, scale=8.0)
    q = queries(2, 8, 64, dtype, scale=8.0)
    for scale in (1.0, -0.5, 0.0):
        check(served, cache, q, dtype, scale=scale, weighted=True)
    sizes = [1e-4, 1.0, 30.0, 0.0] if dtype == "float16" else [1e-20, 1.0, 1e3, 0.0]
    for h, size in enumerate(sizes):
        q[:, 2 * h:2 * h + 2] *= size / 8
    q[0, 3, 5:] *= 2.0 ** -20   # one value far above its head's others
    check(served, cache, q, dtype, scale=0.1)


@pytest.mark.parametrize("heads", [16, 70, 130])
def test_groups_of_many_heads(served, heads):
    check(served, Cache4([40, 1300], 8, 1, 32), queries(2, heads, 32, "bfloat16"), "bfloat16", weighted=True)


def test_results_repeat_bit_for_bit(served):
    import torch
    cache = Cache4([1500, 2700], 16, 2, 128)
    q = queries(2, 8, 128, "bfloat16")
    runs = []
    for _ in range(2):
        w = torch.zeros(2, 2, cache.table.shape[1] * 16, device="cuda")
        runs.append((served.paged_attention(q, cache.keys, cache.values, cache.table, cache.lengths, weights=w), w))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])


@pytest.mark.parametrize("kv, dim, page, lengths, budget, sinks, recent", [
    (2, 64, 16, [200, 0, 40, 41, 90], 40, 4, 8), (1, 96, 7, [61, 100], 30, 0, 0), (3, 32, 1, [70], 9, 4, 5),
    (2, 128, 32, [300, 20], 299, 64, 20)])
def test_evict_4_bits(served, kv, dim, page, lengths, budget, sinks, recent):
    import torch
    cache = Cache4(lengths, page, kv, dim)
    capacity = cache.table.shape[1] * page
    rng = np.random.default_rng(4)
    weights = rng.random((len(lengths), kv, capacity)).astype(np.float32)
    pages = -(-min(budget, capacity) // page)
    target = torch.tensor(rng.permutation(len(lengths) * pages).reshape(len(lengths), pages).astype(np.int32)).cuda()
    pools = [torch.full((len(lengths) * pages, kv, page, dim * 5 // 8), 7, dtype=torch.uint8, device="cuda").permute(0, 2, 1, 3)
             for _ in range(2)]
    kept, new_lengths, new_weights = served.evict_pages(
        cache.keys, cache.values, cache.table, cache.lengths, torch.tensor(weights).cuda(), target, budget=budget,
        sinks=sinks, recent=recent, target_keys=pools[0], target_values=pools[1])
    for s, n in enumerate(lengths):
        held = cache.rows(s, range(n))
        for h in range(kv):
            rows = ref.evict(weights[s, h], n, budget, sinks, recent)
            assert kept[s, h].tolist() == rows + [-1] * (budget - len(rows))
            for pool, source in zip(pools, held):
                moved = pool[target[s].long()].reshape(pages * page, kv, -1)[:, h].cpu().numpy()
                np.testing.assert_array_equal(moved[:len(rows)], source[rows, h])
                assert (moved[len(rows):] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("split", [False, True])
def test_serving_from_4_bits(served, dtype, split):
    """Two prompts in two chunks, decoded tokens with their weights, an eviction, decoding on, scores of the logits: the
    rotated rows go to 4-bit pages, later chunks and tokens see what those hold."""
    import torch
    heads, kv, dim, page, prompts, cut, steps = 8, 2, 64, 16, [70, 41], [50, 10], 5
    rng = np.random.default_rng(5)
    kind = torch_type(dtype)
    rows = [[torch.tensor(rng.normal(size=(n + steps + 1, h, dim))).to(kind).cuda() for h in (heads, kv, kv)] for n in prompts]
    f = frequencies(32)
    pool = [torch.full((24, kv, page, 40), 255, dtype=torch.uint8, device="cuda").permute(0, 2, 1, 3) for _ in range(2)]
    table = torch.arange(12, dtype=torch.int32, device="cuda").reshape(2, 6)
    turned = [[packed.turned32(x.float().cpu().numpy(), np.arange(len(x)), f.cpu().numpy(), split) for x in r[:2]] for r in rows]
    held = [[packed.unpacked(packed.packed(t[1])), packed.unpacked(packed.packed(r[2].float().cpu().numpy()))]
            for t, r in zip(turned, rows)]
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    for begin, end in ((np.zeros(2, int), np.array(cut)), (np.array(cut), np.array(prompts))):
        lengths += torch.tensor(end - begin, dtype=torch.int32, device="cuda")
        offsets = offsets_of(end - begin)
        q, k, v = (torch.cat([r[i][a:b] for r, a, b in zip(rows, begin, end)]) for i in range(3))
        q = served.append_rotated(k, v, *pool, table, lengths, f, offsets, query=q, split_half=split)
        keys, values = (torch.empty(int(end.sum()), kv, dim, device="cuda", dtype=kind) for _ in range(2))
        served.read_pages(*pool, table, lengths, offsets_of(end), keys, values)
        out = served.window_attention(q, keys, values, offsets, offsets_of(end))
        at = 0
        for s, (a, b) in enumerate(zip(begin, end)):
            # the turned queries and the rows read are rounded to the type: taken as they are
            kk, vv = (wide(torch.tensor(x[:b]).to(kind)) for x in held[s])
            want, _, mixed, reach = ref.attend(wide(q[at:at + b - a]), kk, vv, range(a, b), dim ** -0.5)
            bound = ref.output_bound(want, mixed, reach, dim, b, dtype, True)
            assert np.all(np.abs(wide(out[at:at + b - a]) - want) <= bound)
            at += b - a
    weights = torch.zeros(2, kv, 96, device="cuda")
    spent = [np.zeros((kv, n + steps)) for n in prompts]

    def step(table, at, weights, kept=None):
        q, k, v = (torch.stack([r[i][n] for r, n in zip(rows, at)]) for i in range(3))
        q = served.append_rotated(k, v, *pool, table, lengths, f, query=q, split_half=split,
                                  positions=torch.tensor(at, dtype=torch.int32, device="cuda"))
        return q, served.paged_attention(q, *pool, table, lengths, weights=weights)

    for i in range(steps):
        lengths += 1
        q, out = step(table, [n + i for n in prompts], weights)
        for s, n in enumerate(prompts):
            at = n + i
            want, w, mixed, reach = ref.attend(wide(q[s:s + 1]), held[s][0][:at + 1], held[s][1][:at + 1], [at], dim ** -0.5)
            bound = ref.output_bound(want, mixed, reach, dim, at, dtype, False)
            bound = bound + operand_error(wide(q[s:s + 1]), held[s][0][:at + 1], held[s][1][:at + 1], mixed, reach, dim ** -0.5, dtype)
            assert np.all(np.abs(wide(out[s]) - want[0]) <= bound[0])
            spent[s][:, :at + 1] += w[0].reshape(kv, heads // kv, at + 1).sum(1)
    for s, n in enumerate(prompts):
        np.testing.assert_allclose(weights[s, :, :n + steps].cpu().numpy(), spent[s], rtol=1e-4, atol=1e-6)
    target = torch.arange(12, 18, dtype=torch.int32, device="cuda").reshape(2, 3)
    kept, lengths, weights = served.evict_pages(*pool, table, lengths, weights, target, budget=40, sinks=4, recent=8)
    lengths += 1
    q, out = step(target, [n + steps for n in prompts], weights)
    for s, n in enumerate(prompts):
        for h in range(kv):
            at = [*kept[s, h].tolist(), n + steps]
            group = slice(h * heads // kv, (h + 1) * heads // kv)
            want, _, mixed, reach = ref.attend(wide(q[s:s + 1, group]), held[s][0][at, h:h + 1], held[s][1][at, h:h + 1], [40],
                                               dim ** -0.5)
            bound = ref.output_bound(want, mixed, reach, dim, 41, dtype, False)
            bound = bound + operand_error(wide(q[s:s + 1, group]), held[s][0][at, h:h + 1], held[s][1][at, h:h + 1], mixed, reach,
                                          dim ** -0.5, dtype)
            assert np.all(np.abs(wide(out[s, group]) - want[0]) <= bound[0])
    logits = (out.reshape(2, -1).float() @ torch.tensor(rng.normal(size=(heads * dim, 500)), dtype=torch.float32, device="cuda"))
    logprobs, entropy, ids, best = served.log_probabilities(logits, logits.argmax(1).to(torch.int32), top=3)
    log_p, _, p_bound, _ = packed.log_probabilities(wide(logits))
    assert ids[:, 0].tolist() == logits.argmax(1).tolist() and torch.equal(logprobs, best[:, 0])
    assert np.all(np.abs(wide(logprobs) - log_p.max(1)) <= p_bound.max())


def test_captured_calls_replay_side_by_side(pkg):
    """Two graphs of one backend replayed on two streams at once, and the same calls eagerly."""
    import torch
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    b = pkg.CUDABackend(stream=stream.cuda_stream)
    caches = [Cache4([3000, 1900], 16, 2, 64, seed=s) for s in range(2)]
    qs = [queries(2, 8, 64, "bfloat16", seed=s) for s in range(2)]
    weights = [torch.zeros(2, 2, c.table.shape[1] * 16, device="cuda") for c in caches]
    torch.cuda.synchronize()

    def step(i):
        c = caches[i]
        return b.paged_attention(qs[i], c.keys, c.values, c.table, c.lengths, weights=weights[i])

    graphs, results = [], []
    for i in range(2):
        with torch.cuda.stream(stream):
            step(i)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            results.append(step(i))
        graphs.append(graph)
    for i in range(2):
        qs[i].copy_(queries(2, 8, 64, "bfloat16", seed=20 + i))
        weights[i].zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(stream):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    got = [(r.clone(), w.clone()) for r, w in zip(results, weights)]
    for i in range(2):
        weights[i].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for _ in range(3):
                want = step(i)
        torch.cuda.synchronize()
        assert torch.equal(got[i][0], want) and torch.equal(got[i][1], weights[i])


def test_wrong_arguments_are_named(served, pkg):
    import torch
    cache = Cache4([20], 16, 2, 32)
    q = queries(1, 4, 32, "bfloat16")
    with pytest.raises(pkg.CUDAError, match="query has 64 values a head, the pages 32"):
        served.paged_attention(queries(1, 4, 64, "bfloat16"), cache.keys, cache.values, cache.table, cache.lengths)
    with pytest.raises(pkg.CUDAError, match="of one floating type"):
        served.paged_attention(q, cache.keys, cache.values, cache.table, cache.lengths, out=q.half())
    with pytest.raises(pkg.CUDAError, match="target_keys and target_values must be of one type"):
        pools = [torch.zeros(4, 16, 2, 32, device="cuda") for _ in range(2)]
        served.evict_pages(cache.keys, cache.values, cache.table, cache.lengths, torch.zeros(1, 2, 32, device="cuda"), cache.table,
                           budget=20, target_keys=pools[0], target_values=pools[1])
