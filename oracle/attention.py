"""The 4-bit KV cache and the attention over it and over prompts, in numpy.

Quantization follows its definition in fp32 step by step, so that codes and parameters
can be compared bit for bit; attention is computed in 64 bits.
"""
from __future__ import annotations

import numpy as np

from .grinqh_oracle import round_to_dtype, to_f32 as _to_f32


def to_f32(bits: np.ndarray, dtype: str) -> np.ndarray:
    """uint16 bits of dtype ("bf16" or "f16") -> float32."""
    return _to_f32(bits if dtype == "bf16" else bits.view(np.float16), dtype)


def to_bits(x: np.ndarray, dtype: str) -> np.ndarray:
    """float32 -> the bits of dtype, rounded to nearest even."""
    with np.errstate(over="ignore"):
        return round_to_dtype(x, dtype).view(np.uint16)


def record_bytes(dim: int, group: int) -> int:
    return 16 * dim + 128 * (dim // group)


def quantize(x_bits: np.ndarray, dtype: str, group: int):
    """x_bits uint16 [..., D] (the bits of dtype): codes uint8 [..., D], scale and zero bits [..., D/group]."""
    x = to_f32(x_bits, dtype).astype(np.float32)
    g = x.reshape(*x.shape[:-1], -1, group)
    zero, top = g.min(-1), g.max(-1)
    with np.errstate(all="ignore"):
        scale_bits = to_bits(((top - zero) / np.float32(15)).astype(np.float32), dtype)
        scale = to_f32(scale_bits, dtype).astype(np.float32)
        inv = np.where(scale >= np.float32(2.0**-126), np.float32(1) / scale, np.float32(0)).astype(np.float32)
        u = np.rint(np.clip((g - zero[..., None]) * inv[..., None], 0, 15))
    return u.astype(np.uint8).reshape(x.shape), scale_bits, to_bits(zero, dtype)


def _k_word(d: int, dim: int, group: int) -> int:
    g, r = divmod(d, group)
    return (r // (group // 4)) * (dim // 32) + g * (group // 32) + (r % (group // 4)) // 8


def _v_word(pair: int, d: int, dim: int, group: int) -> int:
    g, r = divmod(d, group)
    return ((r // (group // 8)) ^ (2 * (pair % 4))) * (dim // 32) + g * (group // 32) + (r % (group // 8)) // 4


def write_token(record: np.ndarray, token: int, group: int, k, v) -> None:
    """Put one token's quantized k and v, each (codes [D], scale bits, zero bits), into a record of bytes."""
    dim, ng = len(k[0]), len(k[1])
    for d in range(dim):
        at = 4 * (token * (dim // 8) + _k_word(d, dim, group)) + (d % 8) // 2
        shift = 4 * (d % 2)
        record[at] = (record[at] & (0xF0 >> shift)) | (int(k[0][d]) << shift)
        at = 8 * dim + 4 * ((token // 2) * (dim // 4) + _v_word(token // 2, d, dim, group)) + 2 * (token % 2) + (d % 4) // 2
        record[at] = (record[at] & (0xF0 >> shift)) | (int(v[0][d]) << shift)
    for base, (_, scale, zero) in ((16 * dim, k), (16 * dim + 64 * ng, v)):
        p = np.stack([scale, zero], -1).astype(np.uint16).reshape(-1).view(np.uint8)
        record[base + token * 4 * ng: base + (token + 1) * 4 * ng] = p


def read_tokens(records: np.ndarray, dim: int, group: int, dtype: str):
    """records uint8 [n, record] -> K and V [n * 16, D] in 64 bits."""
    n, ng = records.shape[0], dim // group
    tokens, d = np.arange(16)[:, None], np.arange(dim)[None]
    kw = np.array([_k_word(x, dim, group) for x in range(dim)])[None]
    vw = np.array([[_v_word(t // 2, x, dim, group) for x in range(dim)] for t in range(16)])
    k_at = 4 * (tokens * (dim // 8) + kw) + (d % 8) // 2
    v_at = 8 * dim + 4 * ((tokens // 2) * (dim // 4) + vw) + 2 * (tokens % 2) + (d % 4) // 2
    out = []
    for at, base in ((k_at, 16 * dim), (v_at, 16 * dim + 64 * ng)):
        codes = (records[:, at] >> (4 * (d % 2))) & 15
        par = np.ascontiguousarray(records[:, base:base + 64 * ng]).view(np.uint16).reshape(n, 16, ng, 2)
        with np.errstate(all="ignore"):
            par = to_f32(par, dtype).astype(np.float64)
            codes = codes.reshape(n, 16, ng, group).astype(np.float64)
            out.append((codes * par[..., :1] + par[..., 1:]).reshape(n * 16, dim))
    return out


def attention(q, k, v, scale: float):
    """q [n, heads, D], k, v [m, kv heads, D], float64; query j sees keys 0 .. m - n + j.
    Returns out, lse and, for error bounds, sum p |v| like out and max sum |q| |k| like lse."""
    n, heads, dim = q.shape
    m, kv = k.shape[:2]
    out, lse = np.zeros((n, heads, dim)), np.full((n, heads), -np.inf)
    size, reach = np.zeros((n, heads, dim)), np.zeros((n, heads))
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        for j in range(n):
            seen = m - n + j + 1
            if seen <= 0:
                continue
            s = (kh[:seen] @ q[j, h]) * scale
            top = s.max()
            p = np.exp(s - top)
            total = p.sum()
            p /= total
            out[j, h] = p @ vh[:seen]
            size[j, h] = p @ np.abs(vh[:seen])
            lse[j, h] = top + np.log(total)
            reach[j, h] = (np.abs(kh[:seen]) @ np.abs(q[j, h])).max() * abs(scale)
    return out, lse, size, reach
