"""64-bit CPU oracle of the paged KV cache: 4-bit blocks, append, attention — TEST INFRASTRUCTURE ONLY.

Caches are plain lists of rows here: `rows[b]` = float64 [Hkv, length, D]. The page layout is built and
taken apart by pack_pages / unpack_page, written from its definition: per (page, head) the code bytes of
the page's rows (E2M1, element 2i in the low half), then their scale bytes (E4M3, one per 16 elements).
"""
from __future__ import annotations

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                 for e in range(16) for m in range(8)][:127])


def nearest(x: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the nearest grid value (ascending from 0), the even index on a tie, the last one beyond the grid."""
    hi = np.clip(np.searchsorted(grid, x), 1, len(grid) - 1)
    up, down = grid[hi] - x, x - grid[hi - 1]
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)


def fp4_codes(x: np.ndarray, cache_scale: float = 1.0) -> tuple[np.ndarray, np.ndarray]:
    """(codes [.., D] 0..15, scale codes [.., D/16] 0..127) of float64 values; 127 marks a block with a NaN."""
    b = (np.asarray(x, np.float64) / cache_scale).reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    nan = np.isnan(b).any(-1)
    b = np.where(nan[..., None], 0.0, b)
    scale = nearest(np.minimum(np.abs(b).max(-1), 1e30) / 6, E4M3)
    unit = E4M3[scale][..., None]
    q = nearest(np.where(unit > 0, np.minimum(np.abs(b), 1e30) / np.where(unit > 0, unit, 1), 0.0), E2M1)
    q = q + 8 * ((b < 0) & (unit > 0))
    return q.reshape(x.shape).astype(np.uint8), np.where(nan, 127, scale).astype(np.uint8)


def fp4_values(codes: np.ndarray, scales: np.ndarray, cache_scale: float = 1.0) -> np.ndarray:
    grid = np.append(E4M3, np.nan)
    v = np.where(codes >= 8, -1.0, 1.0) * E2M1[codes % 8]
    return v * np.repeat(grid[scales], 16, -1) * cache_scale


def pack_block(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """[page, D] codes and [page, D/16] scale codes -> the bytes of one (page, head) block."""
    both = codes[:, 0::2] | (codes[:, 1::2] << 4)
    return np.concatenate([both.reshape(-1), scales.reshape(-1)]).astype(np.uint8)


def unpack_block(block: np.ndarray, page: int, d: int) -> tuple[np.ndarray, np.ndarray]:
    both = block[: page * d // 2].reshape(page, d // 2)
    codes = np.empty((page, d), np.uint8)
    codes[:, 0::2], codes[:, 1::2] = both & 15, both >> 4
    return codes, block[page * d // 2:].reshape(page, d // 16)


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray) -> np.ndarray:
    """x [tokens, heads, D], cos/sin [tokens, pairs]: interleaved pairs, elements past the pairs copied."""
    x = np.array(x, np.float64)
    n = 2 * cos.shape[1]
    a, b = x[..., 0:n:2].copy(), x[..., 1:n:2].copy()
    c, s = cos[:, None].astype(np.float64), sin[:, None].astype(np.float64)
    x[..., 0:n:2], x[..., 1:n:2] = a * c - b * s, a * s + b * c
    return x


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, past: int, scale: float, softcap: float = 0.0,
              window: int = 0, slopes: np.ndarray | None = None) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """q [n, Hq, D] at positions past.., k/v [Hkv, past + n, D]. Returns (out [n, Hq, D], sum p|v| like out,
    the largest scale * sum |q||k| over a row's keys [n, Hq]): what error bounds are made of."""
    n, hq, d = q.shape
    group = hq // k.shape[0]
    out, mass, size = np.empty_like(q), np.empty_like(q), np.empty((n, hq))
    for i in range(n):
        pos = past + i
        lo = max(0, pos - window + 1) if window else 0
        for h in range(hq):
            kk, vv = k[h // group, lo:pos + 1], v[h // group, lo:pos + 1]
            x = scale * (kk @ q[i, h])
            size[i, h] = scale * (np.abs(kk) @ np.abs(q[i, h])).max()
            if softcap:
                x = softcap * np.tanh(x / softcap)
            if slopes is not None:
                x = x + float(slopes[h]) * (np.arange(lo, pos + 1) - pos)
                size[i, h] += abs(float(slopes[h])) * (pos - lo)
            p = np.exp(x - x.max())
            p /= p.sum()
            out[i, h], mass[i, h] = p @ vv, p @ np.abs(vv)
    return out, mass, size
