"""The paged cache's operators at the edges of what their description allows: empty batches, extreme scalars, small
weights, infinities in visible rows, waits that give up."""
import numpy as np
import pytest

import paged_reference as ref
from conftest import submodule
from test_gpu_paged import TYPES, Cache, check_paged, check_window, queries, served, wide  # noqa: F401

pytestmark = pytest.mark.gpu


def ints(*values):
    import torch
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- eviction -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lengths", [0, -3])
def test_an_eviction_of_empty_sequences_is_over_before_what_follows_it(served, lengths):
    """No row is copied, so that nothing of the copying kernel has work; what it was launched behind still has to end
    before the next kernels of the stream read its outputs."""
    import torch
    batch, heads, page, budget, room = 16, 64, 8, 4096, 1024
    pool = torch.zeros(4, page, heads, 8, device="cuda", dtype=torch.bfloat16)
    table = torch.zeros(batch, budget // page, dtype=torch.int32, device="cuda")
    target = torch.zeros(batch, room, dtype=torch.int32, device="cuda")
    weights = torch.ones(batch, heads, budget, device="cuda")
    empty = torch.full((batch,), lengths, dtype=torch.int32, device="cuda")
    for _ in range(3):
        kept = torch.full((batch, heads, budget), 7, dtype=torch.int32, device="cuda")
        new_lengths = torch.full((batch,), 7, dtype=torch.int32, device="cuda")
        new_weights = torch.full((batch, heads, room * page), 7.0, device="cuda")
        served.evict_pages(pool, pool.clone(), table, empty, weights, target, budget=budget, sinks=2, recent=3,
                           target_keys=pool.clone(), target_values=pool.clone(), kept=kept, new_lengths=new_lengths,
                           new_weights=new_weights)
        # read back to front: the selection's last writes first
        read = new_weights.flip(0).clone(), kept.flip(0).clone(), new_lengths.clone()
        assert not read[0].any() and (read[1] == -1).all() and not read[2].any()


# ---- prompts ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 8, 12, 11])
def test_windows_up_to_the_largest_number(served, dtype, window):
    # more queries than keys (positions below 0), as many, fewer; windows of more, all and all but one of the keys
    new, keys = [19, 10, 4, 300], [12, 10, 9, 0]
    q, k, v = (queries(n, h, 64, dtype, seed=n) for n, h in ((sum(new), 4), (sum(keys), 2), (sum(keys) + 1, 2)))
    qo, ko = (ints(0, *np.cumsum(x).tolist()) for x in (new, keys))
    got = served.window_attention(q, k, v[:-1], qo, ko, window=window, sinks=1)
    served.finish()
    for s in range(4):
        a, b, c, d = sum(new[:s]), sum(new[:s + 1]), sum(keys[:s]), sum(keys[:s + 1])
        if c == d:
            assert not got[a:b].any()
            continue
        want, _, mixed, reach = ref.attend(wide(q[a:b]), wide(k[c:d]), wide(v[c:d]), range(d - c - b + a, d - c), 0.125,
                                           window, 1)
        assert np.all(np.abs(wide(got[a:b]) - want) <= ref.output_bound(want, mixed, reach, 64, 12, dtype, True))


# ---- waits that give up -------------------------------------------------------------------------------------------
LIMIT_NS = 20_000_000


@pytest.fixture
def faulty(pkg):
    """A backend whose prompt attention can be told not to load its values: those who wait for them give up."""
    import torch
    native = submodule("_native")
    backend = pkg.CUDABackend(stream=torch.cuda.current_stream().cuda_stream)
    native.call("mr_context_set_wait_limit", backend.context, LIMIT_NS)

    def fault(on):
        native.call("mr_context_inject_fault", backend.context, int(on))
    backend.fault = fault
    return backend


@pytest.mark.parametrize("heads, kv, dim, new", [
    (4, 2, 64, [60]),            # one tile of keys
    (4, 2, 128, [300, 0, 9]),
    (5, 1, 128, [1400]),         # long: a CTA for each piece
    (8, 8, 64, [40] * 60),       # several pieces to a CTA
])
def test_a_prompt_whose_waits_give_up_ends_and_says_so(pkg, faulty, heads, kv, dim, new):
    import time
    import torch
    q, k, v = (queries(sum(new), h, dim, "bfloat16", seed=h) for h in (heads, kv, kv))
    offsets = ints(0, *np.cumsum(new).tolist())
    want = faulty.window_attention(q, k, v, offsets)
    faulty.finish()
    for _ in range(2):
        faulty.fault(True)
        begin = time.perf_counter()
        faulty.window_attention(q, k, v, offsets)
        with pytest.raises(pkg.CUDAError, match="gave up") as failure:
            faulty.finish()
        assert failure.value.code == submodule("_native").MR_ERR_TIMEOUT
        assert time.perf_counter() - begin < 10
        faulty.finish()   # told once
        faulty.fault(False)
        assert torch.equal(faulty.window_attention(q, k, v, offsets), want)
        faulty.finish()


def test_wait_limits_have_a_least_value(pkg, faulty):
    with pytest.raises(pkg.CUDAError, match="below 1 ms"):
        submodule("_native").call("mr_context_set_wait_limit", faulty.context, 999_999)


def test_a_wait_that_gave_up_is_reported_where_its_results_are_read_or_used(pkg, faulty):
    import torch
    native = submodule("_native")
    rng = np.random.default_rng(3)
    q, k, v = (faulty.upload_array(rng.normal(size=(40, h, 64)), "bfloat16") for h in (4, 2, 2))
    offsets = faulty.upload_array([0, 40], "int32")
    want = faulty.read_array(faulty.window_attention(q, k, v, offsets))
    cache = Cache([40], 16, 2, 64, "bfloat16", extra=6)
    target, weights = ints(*cache.spare[:1])[None], torch.rand(1, 2, 48, device="cuda")
    one, row = queries(1, 4, 64, "bfloat16"), queries(1, 2, 64, "bfloat16")
    calls = [lambda: faulty.paged_attention(one, cache.keys, cache.values, cache.table, cache.lengths),
             lambda: faulty.append_pages(row, row, cache.keys, cache.values, cache.table, cache.lengths),
             lambda: faulty.evict_pages(cache.keys, cache.values, cache.table, cache.lengths, weights, target, budget=16),
             lambda: faulty.window_attention(q, k, v, offsets),
             lambda: faulty.read_array(q)]
    for call in calls:
        faulty.fault(True)
        bad = faulty.window_attention(q, k, v, offsets)
        faulty.fault(False)
        torch.cuda.synchronize()
        with pytest.raises(pkg.CUDAError, match="gave up") as failure:
            call()
        assert failure.value.code == native.MR_ERR_TIMEOUT
        call()   # told once
        assert np.array_equal(faulty.read_array(faulty.window_attention(q, k, v, offsets)), want)
    faulty.fault(True)
    bad = faulty.window_attention(q, k, v, offsets)
    with pytest.raises(pkg.CUDAError, match="gave up"):   # not waited for before
        faulty.read_array(bad)
    faulty.fault(False)
    faulty.finish()


# ---- one token ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv, lengths", [
    (3, 3, [40, 9]), (10, 1, [40]), (5, 1, [33, 200]), (18, 2, [70]),   # groups that blocks of heads leave room in
    (3, 3, [2600, 900]), (10, 1, [1500]), (9, 3, [3000]), (8, 2, [1500]),   # sequences cut between warps
])
def test_an_infinite_visible_key_and_weights(served, dtype, heads, kv, lengths):
    """A key of -inf where all queries are positive: a score of -inf, a weight of 0, and nothing else about the row."""
    cache = Cache(lengths, 16, kv, 64, dtype)
    q = queries(len(lengths), heads, 64, dtype)
    q[:, :, 7] = q[:, :, 7].abs() + 0.25
    rows = [{3}, {3, 8}][:len(lengths)]
    for s, hidden in enumerate(rows):
        for t in hidden:
            cache.keys[int(cache.table[s, t // 16]), t % 16, :, 7] = float("-inf")
            cache.rows[s][0][t, :, 7] = float("-inf")
    check_paged(served, cache, q, dtype, weighted=True, hidden=rows)
    check_paged(served, cache, q, dtype, 30, 9, weighted=True, hidden=rows)


def one_above_many(n, kv, dim, dtype, at=0, above=17.5):
    """n rows of scores 0 and values 1 but for row `at`, whose score is `above` (queries of it alone, scale 1) and whose
    values are 0; and the weight of each of the others, the outputs and row `at`'s weight in 64 bits."""
    import torch
    kind = getattr(torch, dtype)
    keys = torch.zeros(n, kv, dim, device="cuda", dtype=kind)
    values = torch.ones_like(keys)
    keys[at, :, 0], values[at] = 1, 0
    small = np.exp(-np.float64(above))
    total = 1 + (n - 1) * small
    return keys, values, small / total, (n - 1) * small / total, 1 / total


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, batch, heads, kv, dim", [
    (1000, 2, 8, 2, 64), (1000, 1, 3, 3, 32), (500, 1, 8, 1, 128),   # a quarter of the rows each warp's
    (4096, 40, 40, 40, 64), (2048, 24, 80, 80, 128), (32769, 3, 8, 4, 64),   # many rows a warp, cut and whole
])
def test_many_small_weights_beside_a_large_one(served, dtype, n, batch, heads, kv, dim):
    import torch
    page = 64
    pages = -(-n // page)
    for at in (0, n - 1):
        rows = one_above_many(n, kv, dim, dtype, at)
        keys, values = (torch.zeros(pages * page, kv, dim, device="cuda", dtype=rows[0].dtype) for _ in range(2))
        keys[:n], values[:n] = rows[0], rows[1]
        small, want, large = rows[2:]
        q = torch.zeros(batch, heads, dim, device="cuda", dtype=keys.dtype)
        q[:, :, 0] = 17.5
        weights = torch.zeros(batch, kv, pages * page, device="cuda")
        table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(batch, 1)   # all sequences share the pages
        got = served.paged_attention(q, keys.view(pages, page, kv, dim), values.view(pages, page, kv, dim), table,
                                     ints(*[n] * batch), scale=1.0, weights=weights)
        bound = ref.output_bound(want, want, 17.5, dim, n, dtype, False)
        assert np.abs(wide(got) - want).max() <= bound, (wide(got).min(), wide(got).max(), want, bound)
        error = 2 * ref.score_error(17.5, dim) + 2 * (n + heads) * 2.0 ** -24
        spent = np.full(pages * page, small)
        spent[at], spent[n:] = large, 0
        assert np.all(np.abs(wide(weights) * kv / heads - spent) <= (error + 2.0 ** -23) * spent)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, heads, kv, dim", [(8193, 4, 1, 64), (8193, 8, 8, 128), (1000, 6, 2, 128), (700, 130, 1, 16)])
def test_many_small_weights_in_a_prompt(served, dtype, n, heads, kv, dim):
    """The last queries of a prompt, each with one key far above all others."""
    import torch
    for at in (0, 300, n - 9):
        new = 9 if n > 1000 else n
        keys, values = one_above_many(n, kv, dim, dtype, at)[:2]
        q = torch.zeros(new, heads, dim, device="cuda", dtype=keys.dtype)
        q[:, :, 0] = 17.5
        got = wide(served.window_attention(q, keys, values, ints(0, new), ints(0, n), scale=1.0))
        small = np.exp(-np.float64(17.5))
        for i in range(new):
            seen = n - new + i + 1
            want = 1.0 if seen <= at else (seen - 1) * small / (1 + (seen - 1) * small)
            bound = ref.output_bound(want, want, 17.5, dim, seen, dtype, True)
            assert np.abs(got[i] - want).max() <= bound, (at, i, got[i].min(), got[i].max(), want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("step", [0.9, 1.9, 2.1, 7.9, 8.1])
def test_scores_that_grow_from_tile_to_tile(served, dtype, step):
    """The maximum of every 128 keys `step` powers of two above that of those before: weights at the end of their range."""
    import torch
    rng = np.random.default_rng(2)
    kind = getattr(torch, dtype)
    n, heads, dim = 900, 4, 64
    q = torch.zeros(200, heads, dim, device="cuda", dtype=kind)
    q[:, :, 0] = 1
    k = torch.zeros(n, heads, dim, device="cuda", dtype=kind)
    k[:, :, 0] = (torch.arange(n, device="cuda") // 128 * (step * np.log(2))).to(kind)[:, None]
    v = torch.tensor(rng.normal(size=(n, heads, dim))).to(kind).cuda()
    got = served.window_attention(q, k, v, ints(0, 200), ints(0, n), scale=1.0)
    want, _, mixed, reach = ref.attend(wide(q), wide(k), wide(v), range(n - 200, n), 1.0)
    assert np.all(np.abs(wide(got) - want) <= ref.output_bound(want, mixed, reach, dim, n, dtype, True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, dim", [(5, 64), (9, 128), (3, 104)])
def test_a_prompt_repeats_bit_for_bit_whatever_ran_before_it(served, dtype, heads, dim):
    """Groups that leave rows of a tile over: those hold what the kernel before left there."""
    q, k, v = (queries(n, h, dim, dtype, seed=n) for n, h in ((400, heads), (1500, 1), (1499, 1)))
    k = k[:1499]
    before = [queries(12000, h, dim, dtype, seed=h) for h in (4, 1, 1)]
    got = []
    for size in (0.0, 3000.0, 0.0, 1.0):
        served.window_attention(before[0] * size, *before[1:], ints(0, 12000), window=200)
        got.append(wide(served.window_attention(q, k, v, ints(0, 400), ints(0, 1499))))
    assert all(np.array_equal(got[0], x) for x in got[1:])


@pytest.mark.parametrize("dtype", TYPES)
def test_a_sequence_does_not_see_its_neighbours_queries(served, dtype):
    import torch
    q, k, v = (queries(n, h, 64, dtype, seed=n) for n, h in ((60, 8), (1060, 2), (1061, 2)))
    v = v[:1060]
    got = []
    for factor in (1, 100, float("nan")):
        other = torch.cat([q[:10], q[10:] * factor])
        got.append(wide(served.window_attention(other, k, v, ints(0, 10, 60), ints(0, 1000, 1060))[:10]))
    assert all(np.array_equal(got[0], x) for x in got[1:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-36, -9e-37, 1e-38, -1e-39, 1e-45, 1e-50])
def test_prompts_of_the_smallest_scales(served, dtype, scale):
    # down to float32's smallest number, and what it rounds to 0: all visible keys weigh alike
    check_window(served, dtype, 4, 2, 64, [70, 3], [0, 140], scale=scale)
    check_window(served, dtype, 3, 3, 40, [20], [200], window=33, sinks=2, scale=scale)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("scale", [1e-36, 1e-37, 0.0])
def test_small_scales_of_large_scores(served, dtype, scale):
    check_window(served, dtype, 4, 2, 64, [70], [60], scale=scale, size=2.0 ** 115)


# ---- append -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("length, end", [(-2 ** 31, 2 ** 31 - 1), (-2 ** 31, 2), (-1, 2 ** 31 - 1), (0, 2)])
def test_appending_to_a_length_of_none_writes_nothing(served, length, end):
    # a negative length is 0, whatever the offsets are: no row of the sequence is one of its last
    import torch
    pools = [torch.zeros(3, 8, 2, 64, device="cuda") for _ in range(2)]
    rows = [torch.ones(2, 2, 64, device="cuda") for _ in range(2)]
    served.append_pages(*rows, *pools, ints([0, 1, 2]), ints(length), ints(0, end))
    assert not pools[0].any() and not pools[1].any()


def test_a_budget_of_the_largest_number_keeps_all_rows(served):
    # 8 GB of places for kept rows, all but 20 of them empty
    import torch
    cache = Cache([20], 16, 1, 8, "bfloat16", extra=4)
    kept, lengths, weights = served.evict_pages(cache.keys, cache.values, cache.table, cache.lengths,
                                                torch.rand(1, 1, 32, device="cuda"), ints(*cache.spare[:2])[None],
                                                budget=2 ** 31 - 1, sinks=2 ** 30, recent=2 ** 30 - 1)
    served.finish()
    assert kept.shape == (1, 1, 2 ** 31 - 1) and kept[0, 0, :20].tolist() == list(range(20)) and lengths.tolist() == [20]
    assert int(kept[0, 0, 20:].amax()) == -1 and int(kept[0, 0, 20:].amin()) == -1


@pytest.mark.parametrize("nanoseconds", [600_000_000_001, 2 ** 64 - 1])
def test_wait_limits_have_an_end(pkg, faulty, nanoseconds):
    with pytest.raises(pkg.CUDAError, match="above 10 minutes"):
        submodule("_native").call("mr_context_set_wait_limit", faulty.context, nanoseconds)


# ---- values that take the slow way -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths, heads, kv", [([3000], 2, 1), ([1700, 40, 900], 6, 2), ([500], 10, 1)])
def test_an_infinite_value_leaves_the_other_dims_alone(served, dtype, lengths, heads, kv):
    """One part of a cut sequence is worked out again by rows, and joined with parts that are not."""
    import torch
    cache = Cache(lengths, 16, kv, 64, dtype)
    q = queries(len(lengths), heads, 64, dtype)
    for s, n in enumerate(lengths):
        t = n // 3
        cache.values[int(cache.table[s, t // 16]), t % 16, :, 5] = float("inf")
    weights = torch.zeros(len(lengths), kv, cache.table.shape[1] * 16, device="cuda")
    got = served.paged_attention(q, cache.keys, cache.values, cache.table, cache.lengths, weights=weights)
    rest = [d for d in range(64) if d != 5]
    for s, (k, v) in enumerate(cache.rows):
        n = len(k)
        want, w, mixed, reach = ref.attend(wide(q[s:s + 1]), wide(k), wide(v), [n - 1], 0.125)
        bound = ref.output_bound(want, mixed, reach, 64, n, dtype, False)[0]
        assert np.isinf(wide(got[s])[:, 5]).all()
        assert np.all(np.abs(wide(got[s]) - want[0])[:, rest] <= bound[:, rest])
        spent = w[0].reshape(kv, heads // kv, n).sum(1)
        error = 2 * ref.score_error(reach.max(), 64) + 2 * (n + heads) * 2.0 ** -24 + 2.0 ** -23
        assert np.all(np.abs(wide(weights[s, :, :n]) - spent) <= error * spent + 1e-30)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [300.0, 3000.0, 12000.0])
def test_scores_of_many_millions(served, dtype, size):
    """Scores whose neighbouring 32-bit numbers are further apart than a weight's range: the largest takes all."""
    cache = Cache([700, 90], 16, 2, 64, dtype, scale=size)
    q = queries(2, 8, 64, dtype, scale=size)
    # One weight w is left: w v / w.  The output is rounded; in 16-bit prompts w as well, over the sum of it unrounded.
    step = ref.HALF_STEP[dtype]
    bounds = step, step if dtype == "float32" else (1 + step) ** 2 - 1
    got = wide(served.paged_attention(q, cache.keys, cache.values, cache.table, cache.lengths, scale=1.0))
    prompt = [wide(served.window_attention(q[s:s + 1], *cache.rows[s], ints(0, 1), ints(0, n), scale=1.0)[0])
              for s, n in enumerate((700, 90))]
    for s in range(2):
        k, v, x = wide(cache.rows[s][0]), wide(cache.rows[s][1]), wide(q[s])
        for h in range(8):
            scores = k[:, h // 4] @ x[h]
            order = np.argsort(scores)
            reach = (np.abs(k[:, h // 4]) @ np.abs(x[h])).max()
            assert scores[order[-1]] - scores[order[-2]] > 200 * 2.0 ** -23 * reach + 100   # no two within the scores' error
            for out, bound in zip((got[s][h], prompt[s][h]), bounds):
                assert np.all(np.abs(out - v[order[-1], h // 4]) <= bound * np.abs(v[order[-1], h // 4]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv, lengths", [
    (4, 1, [900, 30]), (8, 2, [400]), (7, 1, [1800]), (16, 1, [926, 3]), (34, 2, [700, 1]), (130, 1, [1200]),
    (51, 3, [20]), (72, 8, [2300, 64]),
])
def test_many_small_weights_added_to_large_ones(served, dtype, heads, kv, lengths):
    """What the heads add to a row is added up before it meets the 100 or so that are there: one rounding of the two."""
    import torch
    cache = Cache(lengths, 16, kv, 64, dtype)
    q = queries(len(lengths), heads, 64, dtype)
    was = torch.tensor(np.random.default_rng(9).uniform(50, 120, (len(lengths), kv, cache.table.shape[1] * 16))).float().cuda()
    weights = was.clone()
    served.paged_attention(q, cache.keys, cache.values, cache.table, cache.lengths, weights=weights)
    for s, (k, v) in enumerate(cache.rows):
        n = len(k)
        _, w, _, reach = ref.attend(wide(q[s:s + 1]), wide(k), wide(v), [n - 1], 0.125)
        spent = w[0].reshape(kv, heads // kv, n).sum(1)
        error = 2 * ref.score_error(reach.max(), 64) + 2 * (n + heads) * 2.0 ** -24
        before, after = wide(was[s]), wide(weights[s])
        assert np.all(np.abs(after[:, :n] - before[:, :n] - spent) <= error * spent + 2.0 ** -24 * (before[:, :n] + 2 * spent))
        assert np.array_equal(after[:, n:], before[:, n:])
