"""The paged cache's operators in float64 on the host, row by row, and the error that a kernel's types allow it."""
import numpy as np

HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}   # a rounding, relative


def sees(p, j, window, sinks):
    return j <= p and (not window or p - j < window or j < sinks)


def attend(q, k, v, positions, scale, window=None, sinks=0, hidden=()):
    """q [n, heads, d] at `positions` over k, v [m, kv heads, d].  Returns outputs, softmax weights [n, heads, m],
    the mix of |v| and the largest |q| . |k| a row's score is summed from (for the bounds)."""
    n, heads, d = q.shape
    m, kv_heads = k.shape[:2]
    out, mixed, reach = np.zeros((n, heads, d)), np.zeros((n, heads, d)), np.zeros((n, heads, 1))
    weights = np.zeros((n, heads, m))
    for i, p in enumerate(positions):
        rows = np.array([j for j in range(min(p + 1, m)) if sees(p, j, window, sinks) and j not in hidden], dtype=int)
        if not len(rows):
            continue
        for h in range(heads):
            kk, vv = k[rows, h * kv_heads // heads], v[rows, h * kv_heads // heads]
            s = kk @ q[i, h] * scale
            e = np.exp(s - s.max())
            w = e / e.sum()
            weights[i, h, rows] = w
            out[i, h], mixed[i, h] = w @ vv, w @ np.abs(vv)
            reach[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * abs(scale)
    return out, weights, mixed, reach


def score_error(reach, dim):
    """A score in 32 bits: dim products added with a relative error of 2^-23 a step (tensor cores cut off, others
    round: 2^-24), the scale and the exponential's factor log2(e) rounded, the exponential itself 2^-21."""
    return (dim + 4) * 2.0 ** -23 * reach + 2.0 ** -21


def output_bound(out, mixed, reach, dim, rows, dtype, rounded_weights):
    """|kernel - out|: the output's rounding; of the mix, weights in error by 2 score errors (numerator and sum) and
    `rows` additions in 32 bits twice (numerator and sum); weights rounded to the type where the kernel does that."""
    part = 2 * score_error(reach, dim) + 2 * (rows + 8) * 2.0 ** -24
    if rounded_weights:
        part = part + HALF_STEP[dtype]
    tiny = 2.0 ** -25 if dtype == "float16" else 0.0   # half a step of float16's smallest values
    return HALF_STEP[dtype] * (np.abs(out) + part * mixed) + part * mixed + tiny + 1e-30


def evict(weights, length, budget, sinks, recent):
    """Rows kept of one head's weights [capacity]."""
    n = length
    if n <= budget:
        return list(range(n))
    first = list(range(min(sinks, n)))
    last = list(range(max(n - recent, len(first)), n))
    middle = range(len(first), n - len(last))
    value = lambda t: -np.inf if np.isnan(weights[t]) else weights[t]   # noqa: E731
    nan_last = lambda t: bool(np.isnan(weights[t]))   # noqa: E731
    chosen = sorted(middle, key=lambda t: (nan_last(t), -value(t), t))[:budget - len(first) - len(last)]
    return sorted(first + chosen + last)
