"""The 4-bit KV cache in 64 bits (test oracle, numpy; no counterpart in the reference).

Its definition: groups of 16 dims hold one e4m3 scale s and e2m1 codes; with g a power of two
  s = e4m3(min(max|x / g| / 6, 448)),  code = e2m1(x / g / s),  value = g * s * code,
rounded to nearest, ties to the even code; codes 0 where s is 0, a NaN makes its group NaN.
A page of one layer's K or V is [kv_heads][block * 64 code bytes, block * 8 scale bytes].
Rounding here is a search in the list of representable magnitudes, with no use of the
hardware's or torch's narrow types.
"""
from __future__ import annotations

import numpy as np

GROUP, D, ROW = 16, 128, 72
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                 for e in range(16) for m in range(8)][:127])   # the 128th pattern is NaN


def nearest(x: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the grid value nearest to each x >= 0 (ties: the even index; past the end: the last)."""
    hi = np.clip(np.searchsorted(grid, x), 1, len(grid) - 1)
    lo = hi - 1
    below, above = x - grid[lo], grid[hi] - x
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return np.where(up, hi, lo)


def quantise(x: np.ndarray, g: float = 1.0) -> tuple[np.ndarray, np.ndarray]:
    """Codes [.., 128] (0..15) and scale bytes [.., 8] of rows x [.., 128]."""
    y = np.asarray(x, np.float64).reshape(*x.shape[:-1], D // GROUP, GROUP) / g
    top = np.abs(y).max(-1)
    bad = np.isnan(top)
    scale = np.where(bad, 127, nearest(np.where(bad, 0, np.minimum(top, 1e300)) / 6, E4M3)).astype(np.uint8)
    s = E4M3[np.where(bad, 0, scale)][..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(s > 0, np.minimum(np.abs(y), 1e300) / s, 0)
    codes = nearest(np.nan_to_num(q, nan=0.0), E2M1) + 8 * ((y < 0) & (s > 0))
    return codes.reshape(x.shape).astype(np.uint8), scale


def values(codes: np.ndarray, scale: np.ndarray, g: float = 1.0) -> np.ndarray:
    """Float64 values [.., 128] of codes [.., 128] and scale bytes [.., 8]."""
    v = np.where(codes >= 8, -1.0, 1.0) * E2M1[codes & 7]
    s = np.where((scale & 127) == 127, np.nan, E4M3[np.minimum(scale & 127, 126)])
    return v * np.repeat(s, GROUP, axis=-1) * g


def split_pages(cache: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Codes [pages, heads, block, 128] and scale bytes [pages, heads, block, 8] of uint8 pages."""
    block = cache.shape[-1] // ROW
    packed = cache[..., :block * 64].reshape(*cache.shape[:-1], block, 64)
    codes = np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], D)
    return codes, cache[..., block * 64:].reshape(*cache.shape[:-1], block, 8)


def join_pages(codes: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """The inverse of ``split_pages``."""
    packed = (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)
    lead = codes.shape[:-2]
    return np.concatenate([packed.reshape(*lead, -1), scale.reshape(*lead, -1)], -1)


def store(cache: np.ndarray, rows: np.ndarray, slots, g: float = 1.0) -> np.ndarray:
    """A copy of the pages with rows [N, heads, 128] stored at their slots (-1 skipped)."""
    codes, scale = (a.copy() for a in split_pages(cache))
    block = codes.shape[2]
    c, s = quantise(rows, g)
    for i, slot in enumerate(np.asarray(slots).tolist()):
        if slot >= 0:
            codes[slot // block, :, slot % block] = c[i]
            scale[slot // block, :, slot % block] = s[i]
    return join_pages(codes, scale)


def sequence(cache: np.ndarray, table, n: int, g: float = 1.0) -> np.ndarray:
    """Float64 values [n, heads, 128] of a sequence's first n keys."""
    block = cache.shape[-1] // ROW
    pages = cache[np.asarray(table[: (n + block - 1) // block], dtype=np.int64)]
    v = values(*split_pages(pages), g)                    # [pages, heads, block, 128]
    return v.transpose(0, 2, 1, 3).reshape(-1, cache.shape[1], D)[:n]


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float) -> tuple[np.ndarray, np.ndarray]:
    """Rows q [a, H, 128], the last a of the n positions, over k, v [n, Hk, 128] (causal), in 64
    bits: (output, sum_j p_j |v_j|), both [a, H, 128]; a row that sees no key gives zeros."""
    a, H, _ = q.shape
    n, hk, _ = k.shape
    G = H // hk
    out, size = np.zeros((a, H, D)), np.zeros((a, H, D))
    if n == 0:
        return out, size
    seen = np.arange(n)[None, :] <= (n - a + np.arange(a))[:, None]
    for h in range(H):
        s = np.where(seen, q[:, h].astype(np.float64) @ k[:, h // G].T * scale, -np.inf)
        top = s.max(-1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(top), top, 0))
        total = p.sum(-1, keepdims=True)
        p = p / np.where(total == 0, 1, total)
        out[:, h], size[:, h] = p @ v[:, h // G], p @ np.abs(v[:, h // G])
    return out, size
