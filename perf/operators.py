"""The attention block next to the quantized linears: its cases, plain forms and exact values.

Four operators of a paged cache that holds K and V in 4 bits:

* ``append``  -- quantize new tokens' K and V into the cache, then read them back;
* ``gather``  -- cached tokens as K and V in the model's type;
* ``decode``  -- attention of the last one to few tokens of each sequence over the cache;
* ``prompt``  -- causal attention over packed prompts, whose queries are the last tokens of
  their sequence's keys.

A group of ``group`` channels of a token and head is held as codes u in 0..15 with a scale
and a zero in the model's type: value = scale * u + zero. A cache is a uint8 tensor
[pages, kv heads, page / 16, record]; a record holds 16 tokens of one head:

* K codes, 16 rows of D/2 bytes. Row i is token i; its 32-bit word c * (D/32) + g * (group/32) + j
  holds channels g * group + c * group/4 + 8 j + e at bits 4 e, e = 0..7, c = 0..3;
* V codes, 8 rows of D bytes, a pair of tokens each. Word (c ^ 2 (r % 4)) * (D/32) +
  g * (group/32) + j of row r holds channels g * group + c * group/8 + 4 j + e, c = 0..7,
  e = 0..3: of token 2 r at bits 4 e, of token 2 r + 1 at bits 16 + 4 e;
* the K parameters, 16 x (D/group) x {scale, zero}, then V's.
"""
import functools
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one short prompt arriving alone: latency counts
        dict(name="prompt-short", op="prompt", dtype="bf16", dim=128, heads=32, kv=8, seqs=1, least=77, most=77, prefix=0),
        # a batch of packed prompts of ragged lengths, as a server's prefill step packs them
        dict(name="prompt-packed", op="prompt", dtype="bf16", dim=128, heads=32, kv=8, seqs=14, least=1, most=2048,
             prefix=0),
        # one long prompt on one of four tensor-parallel ranks
        dict(name="prompt-long", op="prompt", dtype="bf16", dim=128, heads=8, kv=2, seqs=1, least=16384, most=16384,
             prefix=0),
        # chunks of prompts whose beginnings are cached already; a smaller model's heads
        dict(name="prompt-chunks", op="prompt", dtype="fp16", dim=64, heads=24, kv=8, seqs=7, least=90, most=700,
             prefix=5000),
        # one user, a short conversation: latency counts
        dict(name="decode-one", op="decode", dtype="bf16", dim=128, heads=32, kv=8, seqs=1, new=1, least=301, most=301,
             page=64, group=128),
        # batch 64 after 512-token prompts, up to 256 tokens generated
        dict(name="decode-batch", op="decode", dtype="bf16", dim=128, heads=32, kv=8, seqs=64, new=1, least=512,
             most=768, page=16, group=64),
        # long documents
        dict(name="decode-long", op="decode", dtype="bf16", dim=128, heads=32, kv=8, seqs=5, new=1, least=50001,
             most=131072, page=64, group=128),
        # four draft tokens per sequence are verified; a smaller model's heads
        dict(name="decode-drafts", op="decode", dtype="fp16", dim=64, heads=24, kv=8, seqs=33, new=4, least=5,
             most=9000, page=32, group=32),
        # a decode step's new tokens enter the cache
        dict(name="append-step", op="append", dtype="bf16", dim=128, kv=8, tokens=64, page=16, group=64),
        # a prefill step's tokens enter the cache
        dict(name="append-prompts", op="append", dtype="fp16", dim=128, kv=8, tokens=16383, page=64, group=128),
        # a cached prefix is read back for the next chunk of its prompt
        dict(name="gather-prefix", op="gather", dtype="bf16", dim=128, kv=8, tokens=1500, page=64, group=128),
        # the prefixes of a batch of chunks
        dict(name="gather-batch", op="gather", dtype="bf16", dim=64, kv=8, tokens=70001, page=32, group=32),
    ]


def _spread(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "decode", "decode", "append", "gather"])
    dim = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), dim=dim, kv=kv)
    if op in ("append", "gather"):
        c.update(tokens=_spread(rng, 1, 16000 if op == "append" else 70000), page=rng.choice([16, 32, 64, 128]),
                 group=rng.choice([g for g in (32, 64, 128) if g <= dim]))
        return c
    c["heads"] = kv * rng.choice([1, 3, 4, 8])
    if op == "decode":
        c["seqs"] = _spread(rng, 1, 100)
        c["new"] = rng.choice([1, 1, 1, 2, 4])
        most = _spread(rng, 2, min(131072, 400000 // c["seqs"]))
        c.update(least=max(1, most // rng.choice([1, 2, 30])), most=most, page=rng.choice([16, 32, 64, 128]),
                 group=rng.choice([g for g in (32, 64, 128) if g <= dim]))
        return c
    c["seqs"] = _spread(rng, 1, 16)
    c["prefix"] = rng.choice([0, 0, _spread(rng, 10, 4000)])
    # pairs of a padded batch stay below those of the long listed prompt
    most = _spread(rng, 1, max(2, int(math.sqrt(8 * 16384**2 / (c["heads"] * c["seqs"]))) - c["prefix"]))
    most = max(1, min(most, 8192))
    c.update(least=max(1, most // rng.choice([1, 2, 30])), most=most)
    return c


def _lens(c):
    """The sequences' (query lengths, key lengths), from the case alone."""
    rng = random.Random("%s %d %d %d" % (c["op"], c["seqs"], c["least"], c["most"]))
    n = [_spread(rng, c["least"], c["most"]) for _ in range(c["seqs"])]
    n[rng.randrange(len(n))] = c["most"]
    if c["op"] == "decode":
        return [c["new"]] * len(n), n
    return n, [x + (rng.randint(0, c["prefix"]) if c["prefix"] else 0) for x in n]


def _pairs(nq, nk):
    """(query, key) pairs that causal attention looks at: query j of n sees m - n + j + 1 keys."""
    return sum(sum(range(max(0, m - n + 1), m + 1)) if m > 0 else 0 for n, m in zip(nq, nk))


def work(c):
    d, kv = c["dim"], c["kv"]
    if c["op"] in ("append", "gather"):
        held, wide = d + 8 * (d // c["group"]), 4 * d  # bytes of a token and head: in the cache, in the model's type
        n = c["tokens"] * kv
        once = n * (held + wide) + 8 * c["tokens"]
        return {"bytes": once * (2 if c["op"] == "append" else 1), "flops": n * d * (12 if c["op"] == "append" else 4)}
    nq, nk = _lens(c)
    rows = sum(nq) * c["heads"]
    io = rows * (2 * 2 * d + 4)
    flops = 4 * d * c["heads"] * _pairs(nq, nk)
    if c["op"] == "decode":
        pages = sum(-(-m // c["page"]) for m in nk)
        return {"bytes": io + sum(nk) * kv * (d + 8 * (d // c["group"])) + 4 * pages + 4 * len(nk), "flops": flops}
    return {"bytes": io + sum(nk) * kv * d * 4 + 8 * (len(nk) + 1), "flops": flops}


# ------------------------------------------------------------------------------ the cache in plain torch
@functools.lru_cache(maxsize=None)
def _places(dim, group, device):
    """Byte of the record that holds channels (2 i, 2 i + 1), and the parameters' bytes: K [16, D/2], V [16, D/2]."""
    words = dim // 32
    ch = torch.arange(0, dim, 2)
    g, r = ch // group, ch % group
    c, s = r // (group // 4), r % (group // 4)
    k_at = (c * words + g * (group // 32) + s // 8) * 4 + (s % 8) // 2
    k = torch.arange(16)[:, None] * (dim // 2) + k_at[None]
    c, s = r // (group // 8), r % (group // 8)
    t = torch.arange(16)[:, None]
    c = c[None] ^ (2 * ((t // 2) % 4))
    v = 8 * dim + (t // 2) * dim + (c * words + (g * (group // 32) + s // 4)[None]) * 4 + (t % 2) * 2 + (s % 4)[None] // 2
    return k.to(device), v.to(device)


def _quantize(x, group):
    """Codes [..., D], scale and zero [..., D/group] of x [..., D]."""
    f = x.float().unflatten(-1, (-1, group))
    zero, top = f.amin(-1), f.amax(-1)
    scale = ((top - zero) / 15.0).to(x.dtype).float()
    inverse = torch.where(scale >= 2.0**-126, 1.0 / scale, torch.zeros_like(scale))
    u = torch.round((f - zero[..., None]) * inverse[..., None]).clamp(0, 15)
    return u.to(torch.uint8).flatten(-2), scale.to(x.dtype), zero.to(x.dtype)


def _plain_append(k, v, cache, slots, group):
    n, kv, dim = k.shape
    page = cache.shape[2] * 16
    ng = dim // group
    at, within = slots // page, slots % page
    flat = cache.view(-1)
    heads = torch.arange(kv, device=k.device)
    record = ((at[:, None] * kv + heads) * cache.shape[2] + (within // 16)[:, None]) * cache.shape[3]  # [n, kv]
    token = within % 16
    for x, places, params in zip((k, v), _places(dim, group, k.device), (16 * dim, 16 * dim + 64 * ng)):
        u, scale, zero = _quantize(x, group)
        flat[record[..., None] + places[token][:, None]] = u[..., 0::2] | (u[..., 1::2] << 4)
        both = torch.stack([scale, zero], -1).contiguous().view(torch.uint8).flatten(2)  # [n, kv, 4 ng]
        where = params + token[:, None] * (4 * ng) + torch.arange(4 * ng, device=k.device)
        flat[record[..., None] + where[:, None]] = both


def _values(codes, params, group):
    """codes uint8 [..., D/2] (two channels a byte), params [..., 2 D/group] -> fp32 [..., D]."""
    u = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (-1, group))
    p = params.float().unflatten(-1, (-1, 2))
    return (u * p[..., :1] + p[..., 1:]).flatten(-2)


def _plain_gather(cache, slots, dim, group, dtype):
    kv, tiles, size = cache.shape[1:]
    ng = dim // group
    at, within = slots // (tiles * 16), slots % (tiles * 16)
    heads = torch.arange(kv, device=cache.device)
    flat = cache.view(-1)
    record = ((at[:, None] * kv + heads) * tiles + (within // 16)[:, None]) * size
    token = within % 16
    out = []
    for places, params in zip(_places(dim, group, cache.device), (16 * dim, 16 * dim + 64 * ng)):
        codes = flat[record[..., None] + places[token][:, None]]
        where = params + token[:, None] * (4 * ng) + torch.arange(4 * ng, device=cache.device)
        out.append(_values(codes, flat[record[..., None] + where[:, None]].view(dtype), group).to(dtype))
    return tuple(out)


def _softmax_v(s, v):
    """softmax(s) @ v and the log of the softmax's sum; rows of -inf alone give 0 and -inf. s is overwritten."""
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
    return out, (total.log() + top).squeeze(-1)


def _plain_decode(q, cache, tables, lens, group, scale):
    b, new, heads, dim = q.shape
    kv, tiles, size = cache.shape[1:]
    ng, page, g = dim // group, tiles * 16, heads // kv
    rec = cache[tables.long()].permute(0, 2, 1, 3, 4).flatten(2, 3)  # [b, kv, n / 16, record]
    n = rec.shape[2] * 16
    parts = []
    for places, at in zip(_places(dim, group, q.device), (16 * dim, 16 * dim + 64 * ng)):
        params = rec[..., at:at + 64 * ng].contiguous().view(q.dtype).unflatten(-1, (16, 2 * ng))
        parts.append(_values(rec[..., places], params, group).flatten(2, 3))  # [b, kv, n, D]
    k, v = parts
    x = q.float().unflatten(2, (kv, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [b, kv, new * g, D]
    s = (x @ k.transpose(-1, -2)).mul_(scale).unflatten(2, (new, g))
    last = lens[:, None].long() - new + torch.arange(new, device=q.device)  # the key of each query's own token
    hidden = torch.arange(n, device=q.device) > last[..., None]
    s = s.masked_fill_(hidden[:, None, :, None], -math.inf).flatten(2, 3)
    out, lse = _softmax_v(s, v)
    out = out.unflatten(2, (new, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return out.to(q.dtype), lse.unflatten(2, (new, g)).permute(0, 2, 1, 3).flatten(2)


def _plain_prompt(q, k, v, cu_q, cu_k, most_q, most_k, scale):
    heads, dim = q.shape[1:]
    kv = k.shape[1]
    g = heads // kv
    device = q.device
    nq, nk = cu_q.diff().long(), cu_k.diff().long()
    iq, ik = torch.arange(most_q, device=device), torch.arange(most_k, device=device)
    rows = (cu_q[:-1, None].long() + iq).clamp(max=q.shape[0] - 1)
    cols = (cu_k[:-1, None].long() + ik).clamp(max=k.shape[0] - 1)
    x = q.float()[rows].unflatten(2, (kv, g)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [b, kv, g * most_q, D]
    key = k.float()[cols].permute(0, 2, 3, 1)
    val = v.float()[cols].permute(0, 2, 1, 3)
    last = (nk - nq)[:, None] + iq
    hidden = (ik > last[..., None]) | (ik >= nk[:, None])[:, None]
    s = (x @ key).mul_(scale).unflatten(2, (g, most_q)).masked_fill_(hidden[:, None, None], -math.inf).flatten(2, 3)
    out, lse = _softmax_v(s, val)
    n = torch.arange(q.shape[0], device=device)
    b = torch.bucketize(n, cu_q[1:].long(), right=True)
    at = n - cu_q.long()[b]
    out = out.unflatten(2, (g, most_q)).flatten(1, 2)[b, :, at]
    lse = lse.unflatten(2, (g, most_q)).flatten(1, 2)[b, :, at]
    return out.to(q.dtype), lse


# ------------------------------------------------------------------------------ what a user's program has in hand
def _tokens(n, kv, dim, dtype, gen):
    """K with channels of different size, as rotary embeddings leave it, and V."""
    size = torch.exp(0.5 * torch.randn(kv, dim, device="cuda", generator=gen))
    k = torch.randn(n, kv, dim, device="cuda", generator=gen).mul_(size).to(dtype)
    v = torch.randn(n, kv, dim, device="cuda", generator=gen).mul_(0.7).to(dtype)
    return k, v


def _filled(pages, c, gen):
    """A cache of `pages` pages with tokens in every place."""
    dim, ng = c["dim"], c["dim"] // c["group"]
    cache = torch.empty(pages, c["kv"], c["page"] // 16, 16 * dim + 128 * ng, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (c["kv"] * c["page"] * dim))
    for p in range(0, pages, step):
        n = (min(pages, p + step) - p) * c["page"]
        k, v = _tokens(n, c["kv"], dim, DTYPES[c["dtype"]], gen)
        _plain_append(k, v, cache, torch.arange(p * c["page"], p * c["page"] + n, device="cuda"), c["group"])
    return cache


def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[c["dtype"]]
    dim, kv = c["dim"], c["kv"]
    if c["op"] in ("append", "gather"):
        # sequences' pages lie anywhere in the cache, tokens of a page in their order
        n, page = c["tokens"], c["page"]
        used = -(-n // page) if c["op"] == "gather" or n > 256 else n
        cache = _filled(used + 3, c, gen)
        where = torch.randperm(used + 3, device="cuda", generator=gen)[:used]
        if used == n:  # a token of each sequence, at any place of its last page
            slots = where * page + torch.randint(page, (n,), device="cuda", generator=gen)
        else:
            slots = (where[:, None] * page + torch.arange(page, device="cuda")).flatten()[:n].contiguous()
        st = dict(op=c["op"], cache=cache, slots=slots, dim=dim, group=c["group"], dtype=dtype)
        if c["op"] == "append":
            st["k"], st["v"] = _tokens(n, kv, dim, dtype, gen)
        return st
    nq, nk = _lens(c)
    scale = dim**-0.5
    if c["op"] == "decode":
        need = [-(-m // c["page"]) for m in nk]
        pages = sum(need) + 3
        cache = _filled(pages, c, gen)
        order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
        tables = torch.zeros(len(nk), max(need), dtype=torch.int32, device="cuda")
        first = 0
        for b, m in enumerate(need):
            tables[b, :m] = order[first:first + m]
            first += m
        q = torch.randn(len(nk), c["new"], c["heads"], dim, device="cuda", generator=gen).to(dtype)
        return dict(op="decode", q=q, cache=cache, tables=tables, group=c["group"], scale=scale,
                    lens=torch.tensor(nk, dtype=torch.int32, device="cuda"))
    cu = [torch.tensor([0] + [sum(n[:i + 1]) for i in range(len(n))], dtype=torch.int32, device="cuda") for n in (nq, nk)]
    if c["prefix"]:
        q = torch.randn(sum(nq), c["heads"], dim, device="cuda", generator=gen).to(dtype)
        k, v = _tokens(sum(nk), kv, dim, dtype, gen)
    else:  # the three parts of a fused projection's output
        k, v = _tokens(sum(nk), kv, dim, dtype, gen)
        q = torch.randn(sum(nq), c["heads"], dim, device="cuda", generator=gen).to(dtype)
        q, k, v = torch.cat([q, k, v], 1).split([c["heads"], kv, kv], 1)
    return dict(op="prompt", q=q, k=k, v=v, cu_q=cu[0], cu_k=cu[1], most_q=max(nq), most_k=max(nk), scale=scale)


@functools.lru_cache(maxsize=None)
def _framework():
    path = os.path.join(os.getcwd(), "vllm-grinqh-plugin_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import grinqh.attention
    return grinqh.attention


def run(s):
    if own:
        f = _framework()
        if s["op"] == "prompt":
            return f.grinqh_prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["scale"])
        if s["op"] == "decode":
            return f.grinqh_kv4_attention(s["q"], s["cache"], s["tables"], s["lens"], s["group"], s["scale"])
        if s["op"] == "append":
            f.grinqh_kv4_append(s["k"], s["v"], s["cache"], s["slots"], s["group"])
        return f.grinqh_kv4_gather(s["cache"], s["slots"], s["group"], s["dtype"])
    if s["op"] == "prompt":
        return _plain_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["most_q"], s["most_k"], s["scale"])
    if s["op"] == "decode":
        return _plain_decode(s["q"], s["cache"], s["tables"], s["lens"], s["group"], s["scale"])
    if s["op"] == "append":
        _plain_append(s["k"], s["v"], s["cache"], s["slots"], s["group"])
    return _plain_gather(s["cache"], s["slots"], s["dim"], s["group"], s["dtype"])


# ------------------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_read(rec, dim, group, dtype):
    """K and V in 64 bits of records [..., record] -> [..., 16, D], by the layout's axes."""
    ng, lead = dim // group, rec.shape[:-1]
    par = rec[..., 16 * dim:].contiguous().view(dtype).double().view(*lead, 2, 16, ng, 1, 2)
    bits = torch.arange(0, 32, 4, device=rec.device)
    words = rec[..., :16 * dim].contiguous().view(torch.int32)
    k = words[..., :2 * dim].reshape(*lead, 16, 4, ng, group // 32, 1)
    k = ((k >> bits) & 15).movedim(-4, -3).reshape(*lead, 16, ng, group).double()
    v = words[..., 2 * dim:].reshape(*lead, 8, 8, ng, group // 32, 1)
    turn = torch.arange(8, device=rec.device)[None] ^ (2 * (torch.arange(8, device=rec.device) % 4))[:, None]
    v = v.gather(-4, turn.view(8, 8, 1, 1, 1).expand(v.shape))
    v = ((v >> bits) & 15).unflatten(-1, (2, 4)).movedim(-2, -5)  # [8 pairs, 2, 8 c, ng, words, 4]
    v = v.movedim(-4, -3).reshape(*lead, 16, ng, group).double()
    out = [x * par[..., i, :, :, :, 0] + par[..., i, :, :, :, 1] for i, x in enumerate((k, v))]
    return [x.flatten(-2) for x in out]


def _exact_attention(q, k, v, scale):
    """q [n, heads, D], k and v [m, kv, D] in 64 bits; query j sees the keys up to m - n + j."""
    n, heads, dim = q.shape
    m, kv = k.shape[:2]
    g = heads // kv
    out, lse = torch.zeros_like(q), q.new_full((n, heads), -math.inf)
    if m == 0:
        return out, lse
    for h in range(kv):
        step = max(1, (1 << 27) // (m * g))
        for a in range(0, n, step):
            z = min(n, a + step)
            s = torch.einsum("ngd,md->ngm", q[a:z, h * g:(h + 1) * g], k[:, h]) * scale
            last = torch.arange(a, z, device=q.device) + (m - n)
            s = s.masked_fill((torch.arange(m, device=q.device) > last[:, None])[:, None], -math.inf)
            part = torch.logsumexp(s, -1)
            lse[a:z, h * g:(h + 1) * g] = part
            p = torch.exp(s - part.clamp(min=-1e300)[..., None])
            out[a:z, h * g:(h + 1) * g] = torch.einsum("ngm,md->ngd", p, v[:, h])
    return out, lse


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "append":
        out = []
        for x in (s["k"], s["v"]):
            f = x.double().unflatten(-1, (-1, c["group"]))
            low, top = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
            scale = ((top - low) / 15).to(x.dtype).double()
            u = torch.where(scale > 0, torch.round((f - low) / scale), torch.zeros_like(f)).clamp(0, 15)
            out.append((scale * u + low).flatten(-2))
        return tuple(out)
    if c["op"] == "gather":
        page = c["page"]
        at, within = s["slots"] // page, s["slots"] % page
        pairs = [_exact_read(s["cache"][at[i:i + 4096], :, within[i:i + 4096] // 16], c["dim"], c["group"], s["dtype"])
                 for i in range(0, c["tokens"], 4096)]
        n = torch.arange(c["tokens"], device="cuda")
        token = within % 16
        return tuple(torch.cat([p[j][torch.arange(p[j].shape[0], device="cuda"), :, token[4096 * i:4096 * (i + 1)]]
                                for i, p in enumerate(pairs)])[n] for j in (0, 1))
    nq, nk = _lens(c)
    outs, lses = [], []
    first_q = first_k = 0
    for b, (n, m) in enumerate(zip(nq, nk)):
        if c["op"] == "decode":
            rec = s["cache"][s["tables"][b, :-(-m // c["page"])].long()].transpose(0, 1).flatten(1, 2)
            k, v = (x.flatten(1, 2)[:, :m].transpose(0, 1) for x in _exact_read(rec, c["dim"], c["group"], s["q"].dtype))
            q = s["q"][b].double()
        else:
            k, v = (s[x][first_k:first_k + m].double() for x in "kv")
            q = s["q"][first_q:first_q + n].double()
        first_q, first_k = first_q + n, first_k + m
        out, lse = _exact_attention(q, k, v, s["scale"])
        outs.append(out)
        lses.append(lse)
    join = torch.stack if c["op"] == "decode" else torch.cat
    return join(outs), join(lses)
