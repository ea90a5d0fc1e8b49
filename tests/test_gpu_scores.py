"""Log probabilities, entropies and most likely tokens against packed_reference.py."""
import numpy as np
import pytest

import packed_reference as ref
from test_gpu_paged import NAN, TYPES, served, torch_type, wide   # noqa: F401

pytestmark = pytest.mark.gpu
INF = float("inf")


def check(served, logits, given=2, top=5, seed=0, **outs):
    import torch
    rows, vocab = logits.shape
    rng = np.random.default_rng(seed)
    tokens = rng.integers(0, vocab, (rows, given)).astype(np.int32)
    if given > 1:
        tokens[0, 1], tokens[-1, 0] = -1, vocab
    got = served.log_probabilities(logits, torch.tensor(tokens).cuda(), top=top, **outs)
    logprobs, entropy, ids, best = got
    assert logprobs.shape == (rows, given) and entropy.shape == (rows,) and ids.shape == best.shape == (rows, top)
    assert logprobs.dtype == entropy.dtype == best.dtype == torch.float32 and ids.dtype == torch.int32
    x = wide(logits)
    log_p, h, p_bound, h_bound = ref.log_probabilities(x)
    index = np.arange(rows)[:, None]
    inside = (tokens >= 0) & (tokens < vocab)
    at = np.where(inside, tokens, 0)
    close(logprobs, np.where(inside, log_p[index, at], 0.0), np.where(inside, p_bound[index, at], 0.0))
    close(entropy, h, h_bound)
    for r in range(rows):
        assert ids[r].tolist() == ref.largest(x[r], top)
    at = ids.cpu().numpy()
    close(best, log_p[index, at], p_bound[index, at])
    return got


def close(got, want, bound):
    got = wide(got)
    with np.errstate(all="ignore"):
        ok = (np.isfinite(want) & (np.abs(got - want) <= bound)) | (got == want) | (np.isnan(got) & np.isnan(want))
    assert ok.all(), (got[~ok][:5], want[~ok][:5], np.broadcast_to(bound, want.shape)[~ok][:5])


def logits_of(rows, vocab, dtype, seed=0, scale=3.0, offset=0.0):
    import torch
    x = np.random.default_rng(seed).normal(size=(rows, vocab)) * scale + offset
    return torch.tensor(x).to(torch_type(dtype)).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, vocab, top", [(1, 1, 1), (3, 2, 2), (2, 7, 7), (5, 33, 20), (1, 128, 128), (7, 512, 20), (3, 1000, 128),
                                              (2, 1031, 64), (300, 515, 3), (4, 2049, 1), (9, 12001, 20)])
def test_small_vocabularies(served, dtype, rows, vocab, top):
    check(served, logits_of(rows, vocab, dtype), 2, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, vocab, top", [(1, 64000, 20), (2, 151937, 128), (40, 32000, 20), (150, 32003, 5), (600, 16384, 0), (1, 9000, 40)])
def test_rows_split_over_ctas_and_whole(served, dtype, rows, vocab, top):
    check(served, logits_of(rows, vocab, dtype, seed=vocab), 3, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [600, 9001, 70001])
@pytest.mark.parametrize("rows", [2, 650])
def test_ties_go_to_the_lowest_token(served, dtype, vocab, rows):
    import torch
    if rows * vocab > 10 ** 7:
        rows = 140
    x = torch.zeros(rows, vocab, device="cuda", dtype=torch_type(dtype))
    check(served, x, 1, 40)                                  # all alike
    check(served, -x, 1, 40)                                 # -0 is 0
    x[:, ::2] = -0.0
    x[0, vocab // 2:] = 1.0                                  # more than half alike and largest
    x[1, -3:] = 2.0
    check(served, x, 1, 40)
    coarse = torch.round(logits_of(rows, vocab, "float32", seed=5)).to(x.dtype)   # few different values
    check(served, coarse, 1, 64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 2000, 65000])
def test_masked_logits(served, dtype, vocab):
    """-inf and the type's lowest value where tokens are not allowed; rows that allow one token, or none."""
    import torch
    lowest = torch.finfo(torch_type(dtype)).min
    for mask in (-INF, lowest):
        x = logits_of(6, vocab, dtype, seed=1)
        x[0, 5:] = mask
        x[1, :-3] = mask
        x[2] = mask
        x[3, torch.randperm(vocab, device="cuda")[:vocab - 20]] = mask
        x[4, 1:] = mask
        got = check(served, x, 2, min(30, vocab))
        if mask == -INF:
            assert (got[3][2] == -INF).all() and got[1][2] == 0
            assert got[2][2].tolist() == list(range(min(30, vocab)))
            assert got[1][4] == 0 and got[3][4, 0] == 0


def test_log_probabilities_of_a_row_of_minus_infinity(served):
    import torch
    x = torch.full((2, 700), -INF, device="cuda")
    x[1, 3] = 2.0
    tokens = torch.tensor([[4, 701], [3, 4]], dtype=torch.int32, device="cuda")
    logprobs, entropy, ids, best = served.log_probabilities(x, tokens, top=3)
    assert logprobs.tolist() == [[-INF, 0.0], [0.0, -INF]] and entropy.tolist() == [0.0, 0.0]
    assert ids.tolist() == [[0, 1, 2], [3, 0, 1]] and best[0].tolist() == [-INF] * 3


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [50, 3001, 66000])
def test_what_is_not_finite(served, dtype, vocab):
    """NaN and +inf reach the row's own results alone; the most likely tokens are still in order."""
    import torch
    x = logits_of(5, vocab, dtype, seed=2)
    x[1, vocab // 3] = NAN
    x[2, vocab // 2] = INF
    x[3] = NAN
    x[4, 2:] = NAN
    logprobs, entropy, ids, best = served.log_probabilities(x, torch.zeros(5, dtype=torch.int32, device="cuda"), top=30)
    assert logprobs.shape == (5,)
    assert torch.isfinite(logprobs[0]) and torch.isnan(logprobs[1:]).all()
    assert torch.isfinite(entropy[0]) and torch.isnan(entropy[1:]).all()
    for r in range(5):
        assert ids[r].tolist() == ref.largest(wide(x[r]), 30)
    assert torch.isfinite(best[0]).all() and torch.isnan(best[1:]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_logits_far_from_zero_and_orders(served, dtype):
    """Differences count, not sizes; falling and rising rows; one token that has all; values to the type's largest."""
    import torch
    top = torch.finfo(torch_type(dtype)).max
    for offset in (-30000.0, 1000.0, 30000.0):
        check(served, logits_of(2, 5000, dtype, scale=offset / 300, offset=offset), 2, 20)
    x = torch.linspace(-20, 20, 66001, device="cuda").to(torch_type(dtype))
    check(served, torch.stack([x, x.flip(0), (x * 50).flip(0), x.abs()]), 2, 128)
    x = logits_of(3, 4000, dtype, seed=4)
    x[0, 17], x[1, 99], x[1, 98], x[2, 5] = 200.0, top, top, -top
    check(served, x, 2, 20)


def test_strided_rows_and_given_outputs(served):
    import torch
    for dtype in TYPES:
        wide_rows = logits_of(6, 4111, dtype)
        for x in (wide_rows[:, 3:4004], wide_rows[::2, 1:], wide_rows[:1].expand(3, -1), wide_rows[1:2, 5:38]):
            check(served, x, 1, 10)
    x = logits_of(4, 900, "bfloat16")
    outs = dict(logprobs=torch.full((4, 6), 7.0, device="cuda")[:, 1:3], entropy=torch.full((8,), 7.0, device="cuda")[::2],
                top_tokens=torch.full((4, 9), 7, dtype=torch.int32, device="cuda")[:, :5],
                top_logprobs=torch.full((4, 9), 7.0, device="cuda")[:, 2:7])
    got = check(served, x, 2, 5, **outs)
    assert got[0] is outs["logprobs"] and got[3] is outs["top_logprobs"]
    assert (got[0]._base[:, 3:] == 7).all() and (got[2]._base[:, 5:] == 7).all() and (got[3]._base[:, 7:] == 7).all()
    assert (got[1]._base[1::2] == 7).all()


def test_only_what_is_asked_for(served, pkg):
    import torch
    x = logits_of(4, 900, "float32")
    logprobs, entropy, ids, best = served.log_probabilities(x)
    assert logprobs is None and ids.shape == best.shape == (4, 0)
    one = served.log_probabilities(x, torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda"), top=2)
    assert one[0].shape == (4,) and torch.equal(one[1], entropy)
    none = served.log_probabilities(x[:0], torch.zeros(0, 2, dtype=torch.int32, device="cuda"), top=4)
    assert [tuple(y.shape) for y in none] == [(0, 2), (0,), (0, 4), (0, 4)]
    for top in (-1, 1.5, True):
        with pytest.raises(ValueError, match="top must be"):
            served.log_probabilities(x, top=top)
    with pytest.raises(pkg.CUDAError, match="at most 128"):
        served.log_probabilities(x, top=129)
    with pytest.raises(ValueError, match="rows, vocabulary"):
        served.log_probabilities(x[0])
    with pytest.raises(ValueError, match="top_tokens must be"):
        served.log_probabilities(x, top=3, top_tokens=ids)


def test_logits_of_the_package(backend):
    rng = np.random.default_rng(3)
    x = rng.normal(size=(3, 500)).astype(np.float32)
    log_p, h, p_bound, h_bound = ref.log_probabilities(x)
    tokens = backend.upload_array([[1], [7], [499]], "int32")
    logprobs, entropy, ids, best = backend.log_probabilities(backend.upload(x), tokens, top=4)
    assert np.all(np.abs(backend.read(logprobs)[:, 0] - log_p[[0, 1, 2], [1, 7, 499]]) <= p_bound.max())
    assert np.all(np.abs(backend.read(entropy) - h) <= h_bound)
    assert backend.read_array(ids).tolist() == [ref.largest(r, 4) for r in x]
    assert backend.log_probabilities(backend.upload(x))[3].shape == (3, 0)


def test_a_captured_and_a_side_streams_call(pkg):
    import torch
    stream = torch.cuda.Stream()
    b = pkg.CUDABackend(stream=stream.cuda_stream)
    x, y = logits_of(3, 70000, "float32"), logits_of(3, 70000, "float32", seed=9)
    want = y.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = b.log_probabilities(x, top=20)
    x.copy_(y)
    torch.cuda.synchronize()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    log_p, h, p_bound, h_bound = ref.log_probabilities(wide(want))
    close(got[1], h, h_bound)
    assert got[2].tolist() == [ref.largest(r, 20) for r in wide(want)]
    again = b.log_probabilities(x, top=20)
    torch.cuda.synchronize()
    assert all(torch.equal(u, w) for u, w in zip(got[1:], again[1:]))   # the same bits each time
