"""Log probabilities of many rows, of which each is a warp's: vocabularies to 1024, and where there are more rows than four an
SM those of up to 32 bytes for each row there is (52 KB in float32, 64 in 16 bits).  A warp has eight of the row's 256 parts a
lane and room for 256 candidates, a fourth of a CTA's.  Against float64 on the GPU: sorts and sums of another path."""
import pytest

from test_gpu_paged import NAN, TYPES, served, torch_type   # noqa: F401
from test_gpu_scores import INF, logits_of

pytestmark = pytest.mark.gpu


def sizes(dtype):
    """The largest vocabularies of each number of rows, one short of them, and a small one."""
    return [(700, 1000), (700, 700 * 8 - 1), (1700, 13312)] if dtype == "float32" else [(700, 1003), (1300, 1300 * 16), (2050, 32768)]


CASES = [(dtype, rows, vocab) for dtype in TYPES for rows, vocab in sizes(dtype)]


def oracle(x):
    """log p [rows, n], the entropy, the order of all tokens, and bounds of both numbers' errors as packed_reference.py has
    them, but of a lane's sums: of each 32 terms 17 follow one another (two sums of 16, added), n / 32 terms a lane, so
    that n / 56 + 64 roundings of 2^-24 hold the lane's and the warp's."""
    import torch
    x = x.double()
    key = torch.nan_to_num(x + 0.0, nan=-INF, posinf=INF, neginf=-1.5e308)   # one zero; NaN behind -inf
    order = torch.sort(-key, dim=1, stable=True).indices
    top = x.amax(1, keepdim=True)
    d = torch.where(torch.isfinite(top), x - top, torch.where(x.isnan() | (x == INF) | top.isnan(), NAN, -INF))
    d = torch.where(top == INF, NAN, d)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    p, far = e / total, torch.where(e > 0, -d, 0.0)
    mean, spread, log_total = (p * far).sum(1), (p * far * far).sum(1), torch.log(total[:, 0])
    log_p, entropy = d - torch.log(total), log_total + mean
    part = 2.0 ** -21 + (x.shape[1] / 56 + 64) * 2.0 ** -24 + 2.0 ** -23 * mean
    p_bound = part[:, None] + 2.0 ** -23 * (d.abs() + log_p.abs() + log_total[:, None])
    h_bound = part * (1 + 2 * mean) + 2.0 ** -23 * (log_total + mean + spread) + 2.0 ** -21 * mean
    none = (x == -INF).all(1)
    log_p[none], entropy[none] = -INF, 0.0
    return log_p, entropy, order, p_bound, h_bound


def close(got, want, bound):
    import torch
    got = got.double()
    ok = (want.isfinite() & ((got - want).abs() <= bound)) | (got == want) | (got.isnan() & want.isnan())
    assert ok.all(), (int((~ok).sum()), got[~ok][:5].tolist(), want[~ok][:5].tolist())
    assert torch.equal(got.isnan(), want.isnan())


def check(served, x, top):
    import torch
    rows, vocab = x.shape
    tokens = torch.randint(0, vocab, (rows, 2), dtype=torch.int32, device="cuda", generator=torch.Generator("cuda").manual_seed(rows))
    got = served.log_probabilities(x, tokens, top=top)
    log_p, entropy, order, p_bound, h_bound = oracle(x)
    close(got[0], log_p.gather(1, tokens.long()), p_bound.gather(1, tokens.long()))
    close(got[1], entropy, h_bound)
    order = order[:, :top]
    assert torch.equal(got[2].long(), order)
    close(got[3], log_p.gather(1, order), p_bound.gather(1, order))
    return got


@pytest.mark.parametrize("dtype, rows, vocab", CASES)
def test_values_and_lists(served, dtype, rows, vocab):
    for top, scale in ((1, 1.0), (20, 3.0), (128, 10.0)):
        check(served, logits_of(rows, vocab, dtype, seed=top, scale=scale), top)


@pytest.mark.parametrize("dtype, rows, vocab", CASES)
def test_masked_rows(served, dtype, rows, vocab):
    """Rows that allow fewer tokens than are asked for, one, or none, beside whole ones; masks of -inf and the lowest value.
    More tokens than a warp's candidates have room for are masked in each."""
    import torch
    for mask in (-INF, torch.finfo(torch_type(dtype)).min):
        x = logits_of(rows, vocab, dtype, seed=1)
        x[0::7, 5:] = mask
        x[1::7, :-3] = mask
        x[2::7] = mask
        x[3::7, torch.randperm(vocab, device="cuda")[:vocab - 20]] = mask
        x[4::7, 1:] = mask
        x[5::7, :-300] = mask
        got = check(served, x, 30)
        if mask == -INF:
            assert (got[2][2::7] == torch.arange(30, device="cuda")).all()
        x[5::7, -300:] = 0.5   # all that are allowed alike, and last
        check(served, x, 128)


@pytest.mark.parametrize("dtype, rows, vocab", CASES)
def test_rows_that_are_not_finite(served, dtype, rows, vocab):
    import torch
    x = logits_of(rows, vocab, dtype, seed=2)
    x[1::6, vocab // 3] = NAN
    x[2::6, vocab // 2] = INF
    x[3::6] = NAN
    x[4::6, 2:] = NAN
    x[5::6, ::2] = NAN
    x[5::6, 1::4] = -INF
    got = check(served, x, 30)
    for r in range(1, 6):
        assert got[0][r::6].isnan().all() and got[1][r::6].isnan().all() and got[3][r::6].isnan().all()
    assert torch.isfinite(got[1][::6]).all()


@pytest.mark.parametrize("dtype, rows, vocab", CASES)
def test_ties(served, dtype, rows, vocab):
    import torch
    x = torch.zeros(rows, vocab, device="cuda", dtype=torch_type(dtype))
    x[::2, ::2] = -0.0
    x[0::5, vocab // 2:] = 1.0
    x[1::5, -3:] = 2.0
    x[2::5] = -7.0
    check(served, x, 40)
    check(served, torch.round(logits_of(rows, vocab, "float32", seed=5)).to(x.dtype), 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_any_start(served, dtype):
    """Rows that start and end off 16-byte boundaries: elements that are no vector's."""
    for start in range(0, 8, 3):
        x = logits_of(640, 2011, dtype, seed=start)
        check(served, x[:, start:2011 - (start * 5) % 7], 20)
