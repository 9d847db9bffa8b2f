"""Attention next to the quantized linears: a paged KV cache held in 4 bits, attention of
a sequence's last tokens over it, and causal attention over packed prompts.

The reference leaves attention to vLLM; these operators are for hosts that own their
decoder layer and want the cache as small as GRINQH's weights. A cache is a uint8 tensor
[pages, kv heads, page_size / 16, record] (``grinqh_kv4_cache``); its layout is in
``include/grinqh_b200.h``. Every function raises on CPU tensors, runs on the current
stream without synchronising, and can be recorded into a CUDA graph. Waits inside the
kernels are bounded (2 s, or ``GRINQH_ATTENTION_WAIT_US``); rows whose wait was lost come
out as NaN, and ``grinqh_check_waits`` raises.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import kernel  # noqa: F401  (loads the op library)
from ._ext import cabi

__all__ = ["grinqh_kv4_cache", "grinqh_kv4_append", "grinqh_kv4_gather", "grinqh_kv4_attention",
           "grinqh_prompt_attention", "grinqh_check_waits"]


def _record_bytes(head_dim: int, group_size: int) -> int:
    return 16 * head_dim + 128 * (head_dim // group_size)


def _head_dim(cache: torch.Tensor, group_size: int) -> int:
    return cache.shape[3] * group_size // (16 * group_size + 128)


@torch.library.register_fake("grinqh::kv4_append")
def _fake_kv4_append(k, v, cache, slots, group_size):
    return None


@torch.library.register_fake("grinqh::kv4_gather")
def _fake_kv4_gather(cache, slots, group_size, dtype):
    shape = (slots.shape[0], cache.shape[1], _head_dim(cache, group_size))
    return cache.new_empty(shape, dtype=dtype), cache.new_empty(shape, dtype=dtype)


@torch.library.register_fake("grinqh::kv4_attention")
def _fake_kv4_attention(q, cache, block_tables, seq_lens, group_size, softmax_scale):
    return q.new_empty(q.shape), q.new_empty(q.shape[:-1], dtype=torch.float32)


@torch.library.register_fake("grinqh::prompt_attention")
def _fake_prompt_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, softmax_scale):
    return q.new_empty(q.shape), q.new_empty(q.shape[:-1], dtype=torch.float32)


_append = torch.ops.grinqh.kv4_append.default
_gather = torch.ops.grinqh.kv4_gather.default
_kv4_attention = torch.ops.grinqh.kv4_attention.default
_prompt_attention = torch.ops.grinqh.prompt_attention.default


def grinqh_kv4_cache(num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64, group_size: int = 128,
                     device="cuda") -> torch.Tensor:
    """An empty cache of ``num_pages`` pages of ``page_size`` tokens (a multiple of 16).
    ``head_dim`` 64 or 128; ``group_size`` channels (32, 64 or 128, at most ``head_dim``)
    share a scale and a zero of the model's type: 4 + 32 / group_size bits a value."""
    if head_dim not in (64, 128) or group_size not in (32, 64, 128) or group_size > head_dim:
        raise ValueError(f"GRINQH: head_dim must be 64 or 128 and group_size 32, 64 or 128, at most head_dim "
                         f"(got {head_dim}, {group_size})")
    if page_size <= 0 or page_size % 16:
        raise ValueError(f"GRINQH: page_size must be a positive multiple of 16 (got {page_size})")
    return torch.zeros(num_pages, num_kv_heads, page_size // 16, _record_bytes(head_dim, group_size),
                       dtype=torch.uint8, device=device)


def grinqh_kv4_append(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor,
                      group_size: int = 128) -> None:
    """Quantize k, v [tokens, kv heads, head_dim] into the cache. ``slots`` (int64) holds
    page * page_size + offset of every token; a slot outside the cache (-1) writes
    nothing, and two tokens of a call must not share one. Views of a fused projection are
    taken as they are. A group that holds a value that is not finite reads back as NaN."""
    _append(k, v, cache, slots, group_size)


def grinqh_kv4_gather(cache: torch.Tensor, slots: torch.Tensor, group_size: int = 128,
                      dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """K and V [tokens, kv heads, head_dim] as the cache holds them at ``slots``, in the
    type that was appended (zeros for a slot outside the cache): a cached prefix for
    ``grinqh_prompt_attention``."""
    return _gather(cache, slots, group_size, dtype)


def grinqh_kv4_attention(q: torch.Tensor, cache: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                         group_size: int = 128,
                         softmax_scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of each sequence's last tokens over the cache: (out like q, lse fp32).

    q [seqs, heads, head_dim], or [seqs, new, heads, head_dim] for several new tokens a
    sequence (drafts to verify); new * heads / kv heads at most 32. ``seq_lens`` (int32)
    counts the new tokens, which have been appended; ``block_tables`` (int32, [seqs,
    width]) lists each sequence's pages. Query j of a sequence of length n sees tokens
    0 .. n - new + j; one that sees none gives zeros and lse = -inf. ``lse`` is the
    natural logarithm of the sum of exp(softmax_scale * q . k). Groups of V whose scale is
    less than 2^-24 of the largest of the sequence and head are summed less exactly."""
    return _kv4_attention(q, cache, block_tables, seq_lens, group_size,
                          q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale)


def grinqh_prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                            cu_seqlens_k: torch.Tensor,
                            softmax_scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Causal attention over packed sequences: (out like q, lse fp32 [tokens, heads]).

    q [tokens, heads, head_dim], k and v [key tokens, kv heads, head_dim], head_dim 64 or
    128; sequence b has rows cu_seqlens_q[b]:cu_seqlens_q[b + 1] of q and
    cu_seqlens_k[b]:cu_seqlens_k[b + 1] of k and v (int32). Its n queries are the last of
    its m tokens: query j sees keys 0 .. m - n + j, so a chunk of a prompt attends its
    cached prefix and itself. A query that sees no key gives zeros and lse = -inf; rows
    of q outside every sequence are left unwritten. Views of a fused projection are taken
    as they are. A key or value that is not finite may reach earlier queries of its own
    sequence (0 * inf is NaN), never another sequence."""
    return _prompt_attention(q, k, v, cu_seqlens_q, cu_seqlens_k,
                             q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale)


def grinqh_check_waits() -> None:
    """Raise if a bounded wait in a kernel of this library on the current device has given up
    since the last check (the rows concerned are then not valid). Synchronises; not during
    a capture."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("GRINQH: grinqh_check_waits synchronises and cannot be captured")
    torch.cuda.synchronize()
    lost = ctypes.c_uint(0)
    if cabi().grinqh_take_error_flags(ctypes.byref(lost)) != 0:
        raise RuntimeError("GRINQH: " + cabi().grinqh_last_error().decode())
    if lost.value:
        raise RuntimeError(f"GRINQH: {lost.value} waits in kernels gave up; rows they concern are not valid")
