"""The 4-bit paged cache in 64 bits: quantisation, record layout and attention, written from the format's definition.

A row of 128 values is four groups of 32 dims, each with a power-of-two scale (one byte, E8M0; 255 is NaN) and
4-bit codes (E2M1).  A record is 16 tokens of one KV head: 1024 code bytes (two codes a byte, the even dim low), then 64
scale bytes.  K: codes [4 groups][16 tokens][16 B], scales [4 groups][16 tokens].  V: codes [4 token quads]
[16 dim octets][4 tokens][4 B], scales [4 token quads][4 groups][4 tokens].
"""

from __future__ import annotations

import math

import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
RECORD = 1088
CODES = 1024


def scale_code(amax: float) -> int:
    """The smallest power of two at which ``amax`` rounds to at most 6 (7 is the tie to 8)."""
    if not math.isfinite(amax):
        return 255
    if amax == 0.0:
        return 1
    mantissa, exponent = math.frexp(amax)  # amax = mantissa 2^exponent, mantissa in [1/2, 1)
    return min(max(exponent - 3 + (mantissa >= 0.875) + 127, 1), 252)


def quantize_row(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes ``[128]``, scale bytes ``[4]``) of one row of 128 float64 values."""
    codes, scales = np.zeros(128, dtype=np.uint8), np.zeros(4, dtype=np.uint8)
    for g in range(4):
        part = x[32 * g:32 * g + 32]
        scales[g] = scale_code(float("nan") if np.isnan(part).any() else float(np.abs(part).max()))
        if scales[g] == 255:
            continue
        mag = np.abs(part) / 2.0 ** (int(scales[g]) - 127)
        distance = np.abs(mag[:, None] - GRID)
        near = distance == distance.min(axis=1, keepdims=True)  # two at a tie: take the even code
        first, last = near.argmax(axis=1), 7 - near[:, ::-1].argmax(axis=1)
        code = np.where(first % 2 == 0, first, last)
        codes[32 * g:32 * g + 32] = code + 8 * np.signbit(part)
    return codes, scales


def values_of(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """float64 ``[128]`` of codes ``[128]`` and scale bytes ``[4]``."""
    s = np.repeat(np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127)), 32)
    return np.where(codes >= 8, -1.0, 1.0) * GRID[codes & 7] * s


def code_at(value: bool, token: int, dim: int) -> int:
    """Byte of the code of (token, dim) in a record."""
    if value:
        return 256 * (token // 4) + 16 * (dim // 8) + 4 * (token % 4) + dim % 8 // 2
    return 256 * (dim // 32) + 16 * token + dim % 32 // 2


def scale_at(value: bool, token: int, group: int) -> int:
    return CODES + (16 * (token // 4) + 4 * group + token % 4 if value else 16 * group + token)


def _maps(value: bool):
    at = np.array([[code_at(value, t, d) for d in range(128)] for t in range(16)])
    sat = np.array([[scale_at(value, t, g) for g in range(4)] for t in range(16)])
    return at, sat


def store(pool: np.ndarray, slot: int, rows: np.ndarray, value: bool) -> None:
    """Writes the quantised ``rows [H_kv, 128]`` of one token into ``pool [blocks of 16, H_kv, 1088]``."""
    at, sat = _maps(value)
    block, token = slot // 16, slot % 16
    for h in range(rows.shape[0]):
        codes, scales = quantize_row(rows[h])
        record = pool[block, h]
        record[at[token, 0::2]] = codes[0::2] | (codes[1::2] << 4)
        record[sat[token]] = scales


def load(pool: np.ndarray, value: bool) -> np.ndarray:
    """float64 ``[blocks, 16, H_kv, 128]`` of a pool ``[blocks of 16, H_kv, 1088]``."""
    at, sat = _maps(value)
    codes = (pool[:, :, at] >> np.where(np.arange(128) % 2, 4, 0).astype(np.uint8)) & 15  # [blocks, H, 16, 128]
    scales = pool[:, :, sat].astype(np.float64)
    s = np.repeat(np.where(scales == 255, np.nan, 2.0 ** (scales - 127)), 32, axis=-1)
    x = np.where(codes >= 8, -1.0, 1.0) * GRID[codes & 7] * s
    return x.transpose(0, 2, 1, 3)


def random_pool(rng: np.random.Generator, blocks: int, heads: int, lo: int = 122, hi: int = 130) -> np.ndarray:
    """A pool of random codes and scales in [lo, hi)."""
    pool = rng.integers(0, 256, (blocks, heads, RECORD), dtype=np.uint8)
    pool[..., CODES:] = rng.integers(lo, hi, (blocks, heads, RECORD - CODES), dtype=np.uint8)
    return pool


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float):
    """One query ``[H, 128]`` over ``k / v [n, H_kv, 128]`` in float64: (out ``[H, 128]``, what the values weigh in
    without their signs, ``sum_t p_t |v_t|``, and per head the largest ``|scale| sum_d |q_d k_td|``)."""
    group = q.shape[0] // k.shape[1]
    k, v = np.repeat(k, group, axis=1), np.repeat(v, group, axis=1)
    s = scale * np.einsum("hd,thd->ht", q, k)
    p = np.exp(s - s.max(axis=1, keepdims=True))
    p /= p.sum(axis=1, keepdims=True)
    size = abs(scale) * np.einsum("hd,thd->ht", np.abs(q), np.abs(k)).max(axis=1)
    return np.einsum("ht,thd->hd", p, v), np.einsum("ht,thd->hd", p, np.abs(v)), size


def table_rows(values: np.ndarray, table, n: int) -> np.ndarray:
    """The first ``n`` rows ``[n, H_kv, 128]`` of a block table over ``values [blocks, 16, H_kv, 128]`` (an id outside
    the pool reads block 0)."""
    ids = [int(b) if 0 <= int(b) < values.shape[0] else 0 for b in table[:-(-n // 16)]]
    return values[ids].reshape(-1, *values.shape[2:])[:n]


def to_torch(pool: np.ndarray, sub: int = 1) -> torch.Tensor:
    """The framework's pool ``[num_blocks, sub, H_kv, 1088]`` of a pool of blocks of 16."""
    return torch.from_numpy(pool.reshape(pool.shape[0] // sub, sub, *pool.shape[1:]).copy())
