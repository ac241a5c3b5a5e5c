"""The 8-bit key/value cache and the attention over it, restated in float64 (test infrastructure).

Held values: blocks of 64 tokens and one head, scale 2^k with the smallest k >= -126 for which the block's largest finite
magnitude is at most 448 * 2^k (e4m3) or 127 * 2^k (int8), k = 0 for a block of zeros; code = round-half-even(x * 2^-k),
a code that would stand for 2^128 replaced by the next lower one, infinities saturated, NaN kept (e4m3) or 0 (int8); masked
tokens are zeros."""
import numpy as np

TOKENS = 64
TOP = {"e4m3": 448.0, "int8": 127.0}


def _round_to_grid(y, dtype):
    if dtype == "int8":
        return np.round(y)
    a = np.abs(y)
    e = np.floor(np.log2(np.maximum(a, 2.0 ** -9)))          # exact here: y is a bf16 value times a power of two
    step = 2.0 ** (np.maximum(e, -6) - 3)
    return np.round(y / step) * step


def held(x, dtype, mask=None):
    """x [n, L, H, 128] float -> the values a cache filled from it stands for, float64.  mask [n, L] or None."""
    x = np.asarray(x, dtype=np.float64).copy()
    if mask is not None:
        x[np.asarray(mask) == 0] = 0.0
    out = np.zeros_like(x)
    n, L, H, _ = x.shape
    for b in range(n):
        for t in range(0, L, TOKENS):
            for h in range(H):
                part = x[b, t:t + TOKENS, h]
                fin = np.abs(part[np.isfinite(part)])
                amax = fin.max() if fin.size else 0.0
                k = 0
                if amax > 0:
                    k = -126
                    if amax > TOP[dtype] * 2.0 ** -126:
                        k = int(np.floor(np.log2(amax / TOP[dtype]))) - 1
                        while amax > TOP[dtype] * 2.0 ** k:
                            k += 1
                y = part / 2.0 ** k
                nan = np.isnan(y)
                top = TOP[dtype]
                if top * 2.0 ** k >= 2.0 ** 128:          # (only where the block holds nearly the largest bf16 values)
                    top = {"e4m3": 240.0, "int8": 63.0}[dtype]
                y = np.clip(np.where(nan, 0.0, y), -top, top)
                y = _round_to_grid(y, dtype) * 2.0 ** k
                out[b, t:t + TOKENS, h] = np.where(nan, np.nan if dtype == "e4m3" else 0.0, y)
    return out


def updated(old, new, start, dtype, mask=None):
    """`old` (held values) after an update with the rows `new` [n, len, H, 128] from token `start` on."""
    out = old.copy()
    end = start + new.shape[1]
    x = old.copy()
    x[:, start:end] = new
    a, b = start // TOKENS * TOKENS, min(old.shape[1], -(-end // TOKENS) * TOKENS)
    out[:, a:b] = held(x[:, a:b], dtype, None if mask is None else mask[:, a:b])
    return out


def attend(q, k, v, mask=None):
    """q [n, n_q, H, 128], k / v [n, L, H, 128] -> (out, spread) [n, n_q, H, 128] float64: the attention and the same sum
    over |v|, by which its rounding errors scale.  Sequences without an unmasked token give zeros."""
    n, n_q, H, d = q.shape
    out, spread = np.zeros((n, n_q, H, d)), np.zeros((n, n_q, H, d))
    for b in range(n):
        keep = np.arange(k.shape[1]) if mask is None else np.nonzero(np.asarray(mask)[b])[0]
        if keep.size == 0:
            continue
        for h in range(H):
            s = q[b, :, h].astype(np.float64) @ k[b, keep, h].astype(np.float64).T / np.sqrt(d)
            p = np.exp(s - s.max(axis=1, keepdims=True))
            p /= p.sum(axis=1, keepdims=True)
            out[b, :, h] = p @ v[b, keep, h]
            spread[b, :, h] = p @ np.abs(v[b, keep, h])
    return out, spread
