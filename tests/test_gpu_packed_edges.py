"""Pages of 4 bits, rotated appends and log probabilities where sizes and callers differ most: tables far longer than their
sequences, pages past 4 GB, several backends at once, chunks whose rows another call has just written."""
import numpy as np
import pytest

import packed_reference as packed
import paged_reference as ref
from test_gpu_packed import Cache4, check, operand_error
from test_gpu_paged import TYPES, queries, served, torch_type, wide   # noqa: F401
from test_gpu_rotated import frequencies, offsets_of
from test_gpu_scores import logits_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [40_000, 140_000, 400_000])
@pytest.mark.parametrize("weighted", [False, True])
def test_tables_longer_than_their_sequences(served, dtype, rows, weighted):
    """What a table could hold chooses how many warps there are; what it holds is a sliver of it."""
    import torch
    cache = Cache4([5000, 3, 0, 700], 16, 2, 64)
    more = torch.full((4, rows // 16 - cache.table.shape[1]), -1, dtype=torch.int32, device="cuda")
    cache.table = torch.cat([cache.table, more], 1)
    check(served, cache, queries(4, 8, 64, dtype), dtype, None, 0, weighted)


def test_attention_over_pages_past_4_gb(served):
    """Pages 2^31 bytes apart, the third past 2^32; rows of a page 2^20 bytes apart."""
    import torch
    store = [torch.empty((1 << 32) + (8 << 20), device="cuda", dtype=torch.uint8) for _ in range(2)]
    pools = [x.as_strided((3, 8, 2, 80), (1 << 31, 1 << 20, 80, 1)) for x in store]
    table = torch.tensor([[2, 0, 1, 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([23], dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(0)
    stored = []
    for pool in pools:
        rows = packed.packed(rng.normal(size=(24, 2, 128)).astype(np.float32))
        pool[torch.tensor([2, 0, 1], device="cuda")] = torch.tensor(rows.reshape(3, 8, 2, 80)).cuda()
        stored.append(packed.unpacked(rows)[:23])
    q = queries(1, 8, 128, "bfloat16")
    got = served.paged_attention(q, *pools, table, lengths)
    want, _, mixed, reach = ref.attend(wide(q), *stored, [22], 128 ** -0.5)
    bound = ref.output_bound(want, mixed, reach, 128, 23, "bfloat16", False)
    bound = bound + operand_error(wide(q), *stored, mixed, reach, 128 ** -0.5, "bfloat16")
    assert np.all(np.abs(wide(got[0]) - want[0]) <= bound[0])


def test_backends_at_once(pkg):
    """Two backends, each on a stream of its own, through the same steps at the same time: the same bits as one alone."""
    import torch
    streams = [torch.cuda.Stream() for _ in range(2)]
    backends = [pkg.CUDABackend(stream=s.cuda_stream) for s in streams]
    lengths, kv, dim, page = [900, 2300, 1], 2, 64, 16
    q, k, v = (queries(sum(lengths), h, dim, "bfloat16", seed=h) for h in (8, kv, kv + 1))
    v = v[:, :kv]
    offsets, f = offsets_of(lengths), frequencies(dim // 2)
    x = logits_of(700, 33001, "float32")

    def steps(b, seed):
        cache = Cache4(lengths, page, kv, dim, seed=seed)
        torch.cuda.synchronize()
        return cache, lambda: run(b, cache)

    def run(b, cache):
        turned = b.append_rotated(k, v, cache.keys, cache.values, cache.table, cache.lengths, f, offsets, query=q)
        rows = b.read_pages(cache.keys, cache.values, cache.table, cache.lengths, offsets, torch.empty_like(k), torch.empty_like(k))
        one = b.paged_attention(turned[torch.tensor([899, 3199, 3200], device="cuda")], cache.keys, cache.values, cache.table,
                                cache.lengths)
        return [turned, *rows, one, *b.log_probabilities(x, top=7)[1:]]

    made = [steps(b, 4) for b in backends]
    results = []
    for _ in range(3):
        for (_, go), stream in zip(made, streams):
            with torch.cuda.stream(stream):
                results.append(go())
    torch.cuda.synchronize()
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@pytest.mark.parametrize("dtype", TYPES)
def test_chunk_after_chunk_reads_what_was_just_written(served, dtype):
    """One prompt in chunks of 1 to 300 tokens, each appended and read back with all before it: the rows read are those that a
    single append of the prompt leaves."""
    import torch
    total, kv, dim, page = 611, 3, 96, 7
    k, v = (queries(total, kv, dim, dtype, seed=s) for s in (1, 2))
    f = frequencies(dim // 2)
    at_once, by_chunks = (Cache4([total], page, kv, dim, seed=9) for _ in range(2))
    served.append_rotated(k, v, at_once.keys, at_once.values, at_once.table, at_once.lengths, f, offsets_of([total]))
    want = served.read_pages(at_once.keys, at_once.values, at_once.table, at_once.lengths, offsets_of([total]),
                             torch.empty_like(k), torch.empty_like(v))
    n = 0
    for new in (1, 7, 300, 2, 33, 268):
        n += new
        lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
        served.append_rotated(k[n - new:n], v[n - new:n], by_chunks.keys, by_chunks.values, by_chunks.table, lengths, f,
                              offsets_of([new]))
        got = served.read_pages(by_chunks.keys, by_chunks.values, by_chunks.table, lengths, offsets_of([n]),
                                torch.empty_like(k[:n]), torch.empty_like(v[:n]))
        assert all(torch.equal(a, b[:n]) for a, b in zip(got, want))
    assert n == total


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, vocab", [(593, 33_003), (1300, 16_500), (1300, 7001), (4100, 1027)])
def test_more_rows_than_run_at_once(served, dtype, rows, vocab):
    """Rows at odd addresses, of which later ones are fetched ahead up to the last: each as if it were alone."""
    import torch
    store = logits_of(rows, vocab + 3, dtype, seed=rows)
    x = store[:, 2:2 + vocab]
    tokens = torch.arange(rows, dtype=torch.int32, device="cuda") % vocab
    got = served.log_probabilities(x, tokens, top=5)
    for r in (0, 1, rows // 2, rows - 1):
        alone = served.log_probabilities(x[r:r + 1], tokens[r:r + 1], top=5)
        assert torch.equal(alone[2][0], got[2][r])
        # sums of the same terms in two orders: a few roundings of 32 bits of numbers below 32
        assert all((a[0] - b[r]).abs().max() <= 64 * 2.0 ** -24 * 32 for a, b in zip((alone[0], alone[1], alone[3]), (got[0], got[1], got[3])))
