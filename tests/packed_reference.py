"""Rotation, 4-bit rows and log probabilities on the host: the header's definitions in NumPy, in 64 bits where the result
is a number to be approached and in 32 where the definition names each rounding."""
import numpy as np

GROUP = 32


def turned32(x, positions, frequencies, split):
    """x [tokens, heads, dim] float32, the first 2 n dims turned: sines rounded once, then products and sums."""
    n = len(frequencies)
    angle = positions.astype(np.float64)[:, None] * frequencies.astype(np.float64)
    cos, sin = np.cos(angle).astype(np.float32)[:, None], np.sin(angle).astype(np.float32)[:, None]
    out = x.astype(np.float32).copy()
    first, second = (slice(0, n), slice(n, 2 * n)) if split else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    a, b = out[..., first].copy(), out[..., second].copy()
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    return out


def turned64(x, positions, frequencies, split):
    """The same in 64 bits, and the sum of the magnitudes that each value is made of."""
    n = len(frequencies)
    angle = (positions.astype(np.float64)[:, None] * frequencies.astype(np.float64))[:, None]
    out, size = x.astype(np.float64).copy(), np.abs(x.astype(np.float64))
    first, second = (slice(0, n), slice(n, 2 * n)) if split else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    z = (out[..., first] + 1j * out[..., second]) * np.exp(1j * angle)
    both = size[..., first] + size[..., second]
    out[..., first], out[..., second] = z.real, z.imag
    size[..., first] = size[..., second] = both
    return out, size


def packed(x):
    """Rows [.., dim] float32 as bytes [.., 5 dim / 8]."""
    with np.errstate(all="ignore"):
        groups = np.asarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
        low, high = groups.min(-1), groups.max(-1)   # NaN if one is
        step = ((high - low) * np.float32(1 / 15)).astype(np.float16)
        base = (low - np.float32(64) * step.astype(np.float32)).astype(np.float16)
        held = np.isfinite(step) & np.isfinite(base)
        code = np.rint((groups - base.astype(np.float32)[..., None]) / step.astype(np.float32)[..., None]) - 64
        code = np.where((held & (step != 0))[..., None], np.clip(code, 0, 15), 0).astype(np.uint8)
    code = code.reshape(x.shape)
    pair = np.stack([np.where(held, step, np.nan), np.where(held, base, np.nan)], -1).astype(np.float16)
    pair = pair.reshape(*x.shape[:-1], x.shape[-1] // 16)
    return np.concatenate([code[..., ::2] | code[..., 1::2] << 4, np.ascontiguousarray(pair).view(np.uint8)], -1)


def unpacked(rows):
    """What bytes [.., 5 dim / 8] stand for, in float64 (the last rounding is to float16)."""
    dim = rows.shape[-1] * 8 // 5
    code = np.stack([rows[..., :dim // 2] & 15, rows[..., :dim // 2] >> 4], -1).reshape(*rows.shape[:-1], dim // GROUP, GROUP)
    pair = np.ascontiguousarray(rows[..., dim // 2:]).view(np.float16).astype(np.float64)
    pair = pair.reshape(*rows.shape[:-1], dim // GROUP, 2)
    with np.errstate(all="ignore"):
        exact = pair[..., :1] * (64.0 + code) + pair[..., 1:]
        return exact.astype(np.float16).astype(np.float64).reshape(*rows.shape[:-1], dim)


def log_probabilities(x):
    """log p [rows, n], the entropy [rows], and bounds of a float32 kernel's errors in both.

    With d = x - max: each e^d is off by 2^-24 (d) + 2^-23 of |d| (its product with log2(e), and that constant) +
    2^-21 (the exponential); sums of n terms by n / 256 + 32 roundings; so S by `part` relative.  log p adds the
    roundings of two differences and of the logarithm.  The entropy's sum has the same errors beside |d|."""
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        top = x.max(1, keepdims=True)
        d = np.where(np.isfinite(top), x - top, -np.inf)
        e = np.exp(d)
        total = e.sum(1, keepdims=True)
        log_p = d - np.log(total)
        p = e / total
        far = np.where(p > 0, -d, 0)
        entropy = np.log(total[:, 0]) + (p * far).sum(1)
        part = 2.0 ** -21 + (x.shape[1] / 256 + 32) * 2.0 ** -24 + 2.0 ** -23 * (p * far).sum(1)
        spread = (p * far * far).sum(1)
        p_bound = part[:, None] + 2.0 ** -23 * (np.abs(d) + np.abs(log_p) + np.log(total)) + 1e-30
        mean = (p * far).sum(1)
        h_bound = part * (1 + 2 * mean) + 2.0 ** -23 * (np.log(total[:, 0]) + mean + spread) + 2.0 ** -21 * mean + 1e-30
    none = np.isneginf(x).all(1)   # the header: -inf and 0
    log_p[none], entropy[none], p_bound[none], h_bound[none] = -np.inf, 0, 0, 0
    return log_p, entropy, p_bound, h_bound


def largest(x, top):
    """Tokens of the `top` largest of a row, falling, the lower of equals first, NaN the lowest."""
    return np.lexsort((np.arange(len(x)), -np.nan_to_num(x, nan=-np.inf, posinf=np.inf, neginf=-np.inf), np.isnan(x)))[:top].tolist()
