"""The attention block of a decoder layer on GRINQH linears and the 4-bit KV cache.

    python -m grinqh.attention_block [--seqs 8] [--prompt 512] [--chunk 256] [--gen 32]
                                     [--max-bits 8] [--page 64] [--group 128]

One layer at the Llama-3-8B shape (hidden 4096, 32 / 8 heads of 128) with random weights,
run as a server would: the prompts' first chunk (packed) through ``grinqh_prompt_attention``,
its K and V into the cache; a second chunk over its prefix read back from the cache; then
tokens one at a time over the cache itself. Prints one JSON line with the times of the
three phases and the cache's size next to a bf16 one. It needs a B200.
"""
from __future__ import annotations

import argparse
import json
import time
from typing import Optional

import torch

from .attention import (grinqh_check_waits, grinqh_kv4_append, grinqh_kv4_attention, grinqh_kv4_cache, grinqh_kv4_gather,
                        grinqh_prompt_attention)
from .kernel import grinqh_gemm_or_gemv
from .utils import pack_codes


class QuantLinear:
    """A random GRINQH linear: symmetric codes with a scale per 128 input channels."""

    def __init__(self, k: int, n: int, max_bits: int, gen: torch.Generator):
        top = 1 << (max_bits - 1)
        codes = torch.randint(-top, top, (k, n), dtype=torch.int8, device="cuda", generator=gen)
        self.packed = pack_codes(codes, max_bits)
        self.scale = torch.full((k // 128, n), 1.7 / (top * k**0.5), dtype=torch.bfloat16, device="cuda")
        self.max_bits, self.n = max_bits, n

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return grinqh_gemm_or_gemv(x, self.packed, self.scale, None, self.max_bits, 128, self.n // 4, [0.0] * 4)


class AttentionBlock:
    """qkv -> rotary embedding -> cache and attention -> o, for ``seqs`` sequences that grow
    together; every sequence's pages lie anywhere in the cache."""

    def __init__(self, seqs: int, max_len: int, hidden: int = 4096, heads: int = 32, kv_heads: int = 8,
                 head_dim: int = 128, max_bits: int = 8, page: int = 64, group: int = 128, seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv, self.dim, self.page, self.group = heads, kv_heads, head_dim, page, group
        self.qkv = QuantLinear(hidden, (heads + 2 * kv_heads) * head_dim, max_bits, gen)
        self.o = QuantLinear(heads * head_dim, hidden, max_bits, gen)
        pages = -(-max_len // page)
        self.cache = grinqh_kv4_cache(seqs * pages, kv_heads, head_dim, page, group)
        self.tables = torch.randperm(seqs * pages, device="cuda", generator=gen).to(torch.int32).view(seqs, pages)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.seqs, self.length = seqs, 0
        half = torch.arange(head_dim // 2, device="cuda", dtype=torch.float32)
        self.freq = 500000.0 ** (-2 * half / head_dim)

    def _rotate(self, x: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        angle = pos[:, None, None].float() * self.freq
        a, b = x.float().chunk(2, -1)
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1).to(x.dtype)

    def _slots(self, first: int, count: int) -> torch.Tensor:
        """Places of tokens first .. first + count of every sequence, sequence by sequence."""
        t = torch.arange(first, first + count, device="cuda")
        return (self.tables[:, t // self.page].long() * self.page + t % self.page).flatten()

    def _count(self, x: torch.Tensor) -> int:
        """New tokens of every sequence in x; their places must be on its pages (an index behind
        them would be a device fault)."""
        count, rest = divmod(x.shape[0], self.seqs)
        if rest or not count:
            raise ValueError(f"GRINQH: {x.shape[0]} rows are not a positive multiple of {self.seqs} sequences")
        if self.length + count > self.tables.shape[1] * self.page:
            raise ValueError(f"GRINQH: {self.length} + {count} tokens do not fit {self.tables.shape[1]} pages of {self.page}")
        return count

    def _project(self, x: torch.Tensor, count: int):
        q, k, v = self.qkv(x).view(-1, self.heads + 2 * self.kv, self.dim).split([self.heads, self.kv, self.kv], 1)
        pos = torch.arange(self.length, self.length + count, device="cuda").repeat(self.seqs)
        return self._rotate(q, pos), self._rotate(k, pos), v

    def prompt(self, x: torch.Tensor) -> torch.Tensor:
        """x [seqs * count, hidden], the next tokens of every sequence, packed: causal over
        themselves and what the cache holds of their prefix."""
        count = self._count(x)
        q, k, v = self._project(x, count)
        ends = torch.arange(self.seqs + 1, dtype=torch.int32, device="cuda")
        keys, values = k, v
        if self.length:
            shape = (self.seqs, -1, self.kv, self.dim)
            before = grinqh_kv4_gather(self.cache, self._slots(0, self.length), self.group, x.dtype)
            keys, values = (torch.cat([b.view(shape), new.reshape(shape)], 1).flatten(0, 1)
                            for b, new in zip(before, (k, v)))
        out, _ = grinqh_prompt_attention(q, keys, values, ends * count, ends * (self.length + count))
        self._append(k, v, count)
        return self.o(out.flatten(1))

    def token(self, x: torch.Tensor) -> torch.Tensor:
        """x [seqs, hidden]: one more token of every sequence, over the cache."""
        if self._count(x) != 1:
            raise ValueError(f"GRINQH: {x.shape[0]} rows, but a token of each of {self.seqs} sequences was expected")
        q, k, v = self._project(x, 1)
        self._append(k, v, 1)
        out, _ = grinqh_kv4_attention(q, self.cache, self.tables, self.lens, self.group)
        return self.o(out.flatten(1))

    def _append(self, k: torch.Tensor, v: torch.Tensor, count: int) -> None:
        grinqh_kv4_append(k, v, self.cache, self._slots(self.length, count), self.group)
        self.length += count
        self.lens += count


def _timed(f) -> float:
    torch.cuda.synchronize()
    t = time.perf_counter()
    f()
    torch.cuda.synchronize()
    return time.perf_counter() - t


def main(argv: Optional[list] = None) -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--seqs", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=512, help="tokens of a prompt's first chunk")
    ap.add_argument("--chunk", type=int, default=256, help="tokens of its second chunk")
    ap.add_argument("--gen", type=int, default=32)
    ap.add_argument("--max-bits", type=int, default=8)
    ap.add_argument("--page", type=int, default=64)
    ap.add_argument("--group", type=int, default=128)
    args = ap.parse_args(argv)
    hidden = 4096
    gen = torch.Generator(device="cuda").manual_seed(1)

    def rows(n):
        return torch.randn(n, hidden, device="cuda", generator=gen).to(torch.bfloat16)

    times = {}
    for _ in range(2):  # the second run is the timed one
        block = AttentionBlock(args.seqs, args.prompt + args.chunk + args.gen, max_bits=args.max_bits, page=args.page,
                               group=args.group)
        first, second = rows(args.seqs * args.prompt), rows(args.seqs * args.chunk)
        steps = [rows(args.seqs) for _ in range(args.gen)]
        times["prompt_ms"] = 1e3 * _timed(lambda: block.prompt(first))
        times["chunk_ms"] = 1e3 * _timed(lambda: block.prompt(second))
        times["token_ms"] = 1e3 * _timed(lambda: [block.token(x) for x in steps]) / max(1, args.gen)
    grinqh_check_waits()
    held = block.cache.numel()
    full = 4 * block.tables.numel() * args.page * block.kv * block.dim
    print(json.dumps({"seqs": args.seqs, "prompt": args.prompt, "chunk": args.chunk, "gen": args.gen,
                      **{k: round(v, 4) for k, v in times.items()}, "cache_mib": round(held / 2**20, 2),
                      "bf16_cache_mib": round(full / 2**20, 2)}))


if __name__ == "__main__":
    main()
