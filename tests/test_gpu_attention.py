"""The 4-bit cache and the attention operators against the numpy oracle on a B200.

Tolerances follow from the types, before any run:
* out: the weights p enter the matrix products in 16 bits (unit roundoff 2^-8 for bf16,
  2^-11 for fp16) and out is rounded once; a score's error d moves every weight by a
  factor e^d. So |out - ref| <= (u_p + 2 d) sum p |v'| + u |ref| + what underflows, with |v'| = |v|
  for prompts and |code * scale| (+ |zero|) for the cache.
* d: products of 16-bit values are exact in fp32; sums of D of them, the scale and the
  base-2 logarithm cost a few units of 2^-22 of the largest sum |q| |k|.
* lse: d and fp32's rounding of a value of its size.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import attention as A  # noqa: E402

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from grinqh import attention as G  # noqa: E402

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"bf16": 2.0**-8, "f16": 2.0**-11}
SHAPES = [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)]


def bits(t):
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


def rand(shape, dtype, seed, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[-1:], generator=g))
    return x.to(DT[dtype]).cuda()


def bounds(dtype, p_unit, size, reach, ref, n):
    d = 2.0**-20 * (reach[..., None] + 1)
    return (p_unit + 2 * d) * size + UNIT[dtype] * np.abs(ref) + n * 2.0**-24 * size.max(initial=0) + 1e-30


def check(got, lse, ref, ref_lse, size, reach, dtype, p_unit, n):
    got, lse = got.double().cpu().numpy(), lse.double().cpu().numpy()
    off = np.abs(got - ref)
    limit = bounds(dtype, p_unit, size, reach, ref, n)
    assert (off <= limit).all(), f"worst {np.max(off / limit)} of the bound"
    none = np.isneginf(ref_lse)
    assert np.array_equal(np.isneginf(lse), none)
    assert (got[none] == 0).all()
    lse, ref_lse, reach = lse[~none], ref_lse[~none], reach[~none]
    assert (np.abs(lse - ref_lse) <= 2.0**-20 * (reach + 1 + np.abs(ref_lse))).all()


# ------------------------------------------------------------------ cache
def slots_for(kind, n, pages, page, seed):
    rng = np.random.default_rng(seed)
    if kind == "anywhere":
        return rng.permutation(pages * page)[:n]
    first = {"aligned": 0, "odd": 3}[kind]
    order = rng.permutation(pages)
    return np.concatenate([p * page + np.arange(page) for p in order])[first:first + n]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim,group", SHAPES)
@pytest.mark.parametrize("tokens,heads,page,kind", [(1, 1, 16, "anywhere"), (37, 3, 48, "anywhere"),
                                                    (64, 2, 16, "aligned"), (45, 2, 32, "odd")])
def test_append_and_gather(dtype, dim, group, tokens, heads, page, kind):
    """Every byte of the cache: the tokens' codes and parameters, and the rest as it was."""
    pages = -(-(tokens + 3) // page) + 1
    slots = slots_for(kind, tokens, pages, page, tokens).copy()
    skip = np.zeros(tokens, bool)
    if tokens > 4:  # padding and places past the end write nothing
        slots[2], slots[4] = -1, pages * page
        skip[[2, 4]] = True
    fused = rand((tokens, 3 * heads, dim), dtype, dim + group)
    k, v = fused[:, heads:2 * heads], fused[:, 2 * heads:]
    g = torch.Generator().manual_seed(3)
    cache = torch.randint(0, 256, (pages, heads, page // 16, A.record_bytes(dim, group)), dtype=torch.uint8, generator=g)
    want = cache.numpy().copy()
    cache = cache.cuda()
    qk, qv = A.quantize(bits(k), dtype, group), A.quantize(bits(v), dtype, group)
    for i, s in enumerate(slots):
        if not skip[i]:
            for h in range(heads):
                A.write_token(want[s // page, h, s % page // 16], s % 16, group, [x[i, h] for x in qk], [x[i, h] for x in qv])
    ts = torch.from_numpy(slots).cuda()
    G.grinqh_kv4_append(k, v, cache, ts, group)
    assert np.array_equal(cache.cpu().numpy(), want)
    gk, gv = G.grinqh_kv4_gather(cache, ts, group, DT[dtype])
    both = [A.read_tokens(want[:, h].reshape(-1, want.shape[-1]), dim, group, dtype) for h in range(heads)]
    for j, got in enumerate((gk, gv)):
        for h in range(heads):
            with np.errstate(all="ignore"):
                ref = A.to_bits(both[h][j][np.where(skip, 0, slots)].astype(np.float32), dtype)
            ref[skip] = 0
            r = torch.from_numpy(ref.view(np.int16).copy()).view(DT[dtype])
            assert torch.equal(got[:, h].cpu(), r)


def test_append_constant_and_not_finite_groups():
    x = torch.randn(4, 1, 128).to(torch.bfloat16)
    x[0] = 1.5
    x[1, 0, 5], x[2, 0, 70], x[3, 0, 127] = math.nan, math.inf, -math.inf
    cache = G.grinqh_kv4_cache(1, 1, 128, 16, 64)
    slots = torch.arange(4).cuda()
    G.grinqh_kv4_append(x.cuda(), x.cuda(), cache, slots, 64)
    for got in G.grinqh_kv4_gather(cache, slots, 64):
        assert (got[0] == 1.5).all()
        bad = got.isnan().view(4, 2, 64).cpu()
        assert bad[1, 0].all() and bad[2, 1].all() and bad[3, 1].all()
        assert not (bad[1, 1].any() or bad[2, 0].any() or bad[3, 0].any())


def test_places_beyond_32_bit_offsets():
    """A cache of more than 4 GB: its last pages are written, read and attended."""
    dim, group, heads, page = 64, 64, 2, 16
    pages = (1 << 32) // (heads * A.record_bytes(dim, group)) + 5
    cache = torch.empty(pages, heads, 1, A.record_bytes(dim, group), dtype=torch.uint8, device="cuda")
    k, v, q = rand((20, heads, dim), "bf16", 1), rand((20, heads, dim), "bf16", 2), rand((1, 4, dim), "bf16", 3)
    tables = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32).cuda()
    slots = (tables.long()[0, torch.arange(20) // 16] * 16 + torch.arange(20, device="cuda") % 16)
    cache[tables[0].long()] = 0
    G.grinqh_kv4_append(k, v, cache, slots, group)
    small = G.grinqh_kv4_cache(2, heads, dim, page, group)
    G.grinqh_kv4_append(k, v, small, torch.arange(20).cuda(), group)
    assert torch.equal(cache[tables[0].long()], small)
    lens = torch.tensor([20], dtype=torch.int32).cuda()
    got = G.grinqh_kv4_attention(q, cache, tables, lens, group)
    want = G.grinqh_kv4_attention(q, small, torch.tensor([[0, 1]], dtype=torch.int32).cuda(), lens, group)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------ attention over the cache
def cache_case(dtype, dim, group, kv, lens, page, seed, spread=0.5):
    """A cache whose unused places hold bytes that read as NaN, tables with entries outside
    the cache behind each sequence's pages, and K, V in 64 bits."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    rng = np.random.default_rng(seed)
    order = rng.permutation(pages)
    width = max(need) + 2
    tables = np.full((len(lens), width), 1 << 30, np.int32)
    cache = torch.full((pages, kv, page // 16, A.record_bytes(dim, group)), 255, dtype=torch.uint8).cuda()
    keys = []
    at = 0
    for b, n in enumerate(lens):
        tables[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        if n:
            t = np.arange(n)
            slots = torch.from_numpy(tables[b, t // page].astype(np.int64) * page + t % page).cuda()
            k, v = rand((n, kv, dim), dtype, seed + 2 * b, spread), rand((n, kv, dim), dtype, seed + 2 * b + 1)
            G.grinqh_kv4_append(k, v, cache, slots, group)
    host = cache.cpu().numpy()
    for b, n in enumerate(lens):
        rec = host[tables[b, :need[b]]]  # [pages, kv, tiles, record]
        kvs = [A.read_tokens(rec[:, h].reshape(-1, rec.shape[-1]), dim, group, dtype) for h in range(kv)]
        keys.append([np.stack([x[i][:n] for x in kvs], 1) for i in (0, 1)])
    return cache, torch.from_numpy(tables).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), keys


def code_size(v, group):
    """|code * scale| + |zero| is at most this for every value of the group."""
    g = np.abs(v.reshape(*v.shape[:-1], -1, group)).max(-1, keepdims=True)
    return np.broadcast_to(3 * g, (*g.shape[:-1], group)).reshape(v.shape)


def check_cached(q, case, group, dtype, scale=None):
    cache, tables, lens, keys = case
    out, lse = G.grinqh_kv4_attention(q, cache, tables, lens, group, scale)
    assert out.shape == q.shape and lse.shape == q.shape[:-1] and lse.dtype == torch.float32
    q4 = q if q.dim() == 4 else q[:, None]
    o4, l4 = out.view(q4.shape), lse.view(q4.shape[:-1])
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    for b, (k, v) in enumerate(keys):
        x = q4[b].double().cpu().numpy()
        ref, ref_lse, _, reach = A.attention(x, k, v, scale)
        size = A.attention(x, k, code_size(v, group), scale)[2] if len(k) else np.zeros_like(ref)
        kr = np.abs(k).max(initial=0) * np.abs(x).sum(-1) * abs(scale) * 3  # codes reach 3 x the largest |k|
        check(o4[b], l4[b], ref, ref_lse, size, np.maximum(reach, kr), dtype, 2.0**-11, len(k))
    return out, lse


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim,group", SHAPES)
@pytest.mark.parametrize("heads,kv,new,page", [(1, 1, 1, 16), (8, 2, 1, 64), (6, 2, 2, 32), (8, 1, 4, 48), (9, 1, 3, 16),
                                               (24, 1, 1, 128)])
def test_cached_attention(dtype, dim, group, heads, kv, new, page):
    lens = [0, 1, 2, 15, 16, 17, 33, 100, 257]
    case = cache_case(dtype, dim, group, kv, lens, page, dim + heads + new)
    q = rand((len(lens), new, heads, dim), dtype, 5, 0.3)
    check_cached(q if new > 1 else q[:, 0], case, group, dtype)


@pytest.mark.parametrize("lens", [[5000], [3, 2100, 1], [1300] * 3 + [0] * 30 + [700]])
@pytest.mark.parametrize("dim,group,heads,kv,new", [(128, 128, 8, 2, 1), (64, 32, 3, 1, 4)])
def test_cached_attention_long(lens, dim, group, heads, kv, new):
    """Rows whose tokens are split over many blocks, next to rows with few or none."""
    case = cache_case("bf16", dim, group, kv, lens, 64, sum(lens))
    check_cached(rand((len(lens), new, heads, dim), "bf16", 6, 0.3), case, group, "bf16")


@pytest.mark.parametrize("dtype,limit", [("bf16", 3e-3), ("f16", 1e-3)])
def test_cached_attention_long_and_flat(dtype, limit):
    """Nearly equal weights over 131071 tokens: out is 1/900 of the codes' sum and the
    zeros' that make it up, so what rounding costs those sums shows. In the 2-norm, relative to out:
    out's own rounding 1.7e-3 (bf16) or 2.1e-4, the weights' 11 bits 7e-4 (2.5e-4 where the middle code is
    given back), fp32 sums 900 x 2^-24 x the square root of the 64 steps of a run: 4.5e-4."""
    n, page = 131071, 64
    cache = G.grinqh_kv4_cache(2048, 1, 128, page, 128)
    k, v = rand((n, 1, 128), dtype, 1), rand((n, 1, 128), dtype, 2, 0.0)
    G.grinqh_kv4_append(k, v, cache, torch.arange(n).cuda(), 128)
    q = rand((1, 4, 128), dtype, 3) * 0.05
    out, lse = G.grinqh_kv4_attention(q, cache, torch.arange(2048, dtype=torch.int32).cuda()[None],
                                      torch.tensor([n], dtype=torch.int32).cuda(), 128)
    kr, vr = (x[:n, None] for x in A.read_tokens(cache.cpu().numpy().reshape(-1, cache.shape[-1]), 128, 128, dtype))
    ref, ref_lse, _, _ = A.attention(q.double().cpu().numpy(), kr, vr, 128**-0.5)
    assert np.linalg.norm(out.double().cpu().numpy() - ref) <= limit * np.linalg.norm(ref)
    assert np.abs(lse.double().cpu().numpy() - ref_lse).max() <= 2.0**-20 * (1 + np.abs(ref_lse).max())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_cached_attention_large_scores(dtype):
    """Scores of hundreds that rise along the sequence, and values of very different size."""
    case = cache_case(dtype, 128, 64, 1, [700, 40], 16, 11, spread=1.2)
    q = rand((2, 4, 128), dtype, 8, 1.0) * 4
    check_cached(q, case, 64, dtype, 0.5)


def test_cached_attention_small_and_large_values():
    """V of 1e-6 and of 1e4 in bf16: the weights' 16-bit range must follow the scales."""
    for size in (1e-6, 1e4):
        cache, tables, lens, keys = cache_case("bf16", 128, 128, 1, [300], 16, 21)
        k, v = rand((300, 1, 128), "bf16", 1), rand((300, 1, 128), "bf16", 2) * size
        t = torch.arange(300).cuda()
        G.grinqh_kv4_append(k, v, cache, tables[0].long()[t // 16] * 16 + t % 16, 128)
        rec = cache.cpu().numpy()[tables[0, :19].cpu().numpy()][:, 0].reshape(-1, cache.shape[-1])
        keys = [[x[:300, None] for x in A.read_tokens(rec, 128, 128, "bf16")]]
        check_cached(rand((1, 4, 128), "bf16", 3), (cache, tables, lens, keys), 128, "bf16")


def test_cached_attention_views_stream_and_graph():
    case = cache_case("bf16", 128, 128, 2, [300, 77], 32, 31)
    cache, tables, lens, _ = case
    fused = rand((2, 16, 128), "bf16", 9)
    want = check_cached(fused[:, 4:12].contiguous(), case, 128, "bf16")
    wide = torch.zeros(2, 4 * tables.shape[1], dtype=torch.int32, device="cuda")
    wide[:, :tables.shape[1]] = tables
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = G.grinqh_kv4_attention(fused[:, 4:12], cache, wide[:, :tables.shape[1]], lens, 128)
        again = G.grinqh_kv4_attention(fused[:, 4:12], cache, wide[:, ::1], lens, 128)
    side.synchronize()
    for x in (got, again):
        assert torch.equal(x[0], want[0]) and torch.equal(x[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = G.grinqh_kv4_attention(fused[:, 4:12], cache, tables, lens, 128)
    for _ in range(3):
        kept[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept[0], want[0]) and torch.equal(kept[1], want[1])


def test_cached_attention_is_deterministic():
    cache, tables, lens, _ = cache_case("bf16", 128, 64, 2, [4000, 9, 1200], 64, 41)
    q = rand((3, 8, 128), "bf16", 9)
    first = G.grinqh_kv4_attention(q, cache, tables, lens, 64)
    for _ in range(5):
        again = G.grinqh_kv4_attention(q, cache, tables, lens, 64)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_cached_attention_cuts_lengths_to_the_table():
    cache, tables, lens, keys = cache_case("bf16", 64, 64, 1, [64], 16, 51)
    q = rand((1, 2, 64), "bf16", 9)
    want = G.grinqh_kv4_attention(q, cache, tables[:, :4], lens, 64)
    got = G.grinqh_kv4_attention(q, cache, tables[:, :4], lens + 1000, 64)
    none = G.grinqh_kv4_attention(q, cache, tables[:, :4], lens - 100, 64)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (none[0] == 0).all() and torch.isneginf(none[1]).all()


# ------------------------------------------------------------------ attention over prompts
def prompt_case(nq, nk, heads, kv, dim, dtype, seed, gap=0):
    """Packed q, k, v with `gap` rows of NaN between the sequences of k and v."""
    cu_q = np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)
    cu_k = np.concatenate([[0], np.cumsum(nk)]).astype(np.int32)
    return (rand((int(cu_q[-1]), heads, dim), dtype, seed, 0.3), rand((int(cu_k[-1]), kv, dim), dtype, seed + 1, 0.3),
            rand((int(cu_k[-1]), kv, dim), dtype, seed + 2), torch.from_numpy(cu_q).cuda(), torch.from_numpy(cu_k).cuda())


def check_prompt(q, k, v, cu_q, cu_k, dtype, scale=None, only=None):
    out, lse = G.grinqh_prompt_attention(q, k, v, cu_q, cu_k, scale)
    assert out.shape == q.shape and lse.shape == q.shape[:-1] and lse.dtype == torch.float32
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    x, y, z = (t.double().cpu().numpy() for t in (q, k, v))
    a, b = cu_q.tolist(), cu_k.tolist()
    for i in range(len(a) - 1) if only is None else only:
        r = A.attention(x[a[i]:a[i + 1]], y[b[i]:b[i + 1]], z[b[i]:b[i + 1]], scale)
        check(out[a[i]:a[i + 1]], lse[a[i]:a[i + 1]], *r, dtype, UNIT[dtype], b[i + 1] - b[i])
    return out, lse


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 2), (4, 1), (3, 1), (6, 2)])
def test_prompt_lengths(dtype, dim, heads, kv):
    n = [1, 0, 2, 127, 128, 129, 64, 255, 256, 300]
    check_prompt(*prompt_case(n, n, heads, kv, dim, dtype, heads + dim), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim,heads,kv", [(128, 4, 1), (64, 3, 1), (128, 2, 2)])
def test_prompt_after_prefix_and_without_keys(dtype, dim, heads, kv):
    """Queries at the end of longer keys, more queries than keys, no keys, no queries."""
    nq = [3, 130, 1, 200, 40, 0, 257, 129]
    nk = [260, 131, 400, 70, 0, 50, 257, 128]
    check_prompt(*prompt_case(nq, nk, heads, kv, dim, dtype, dim), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim,heads,kv", [(128, 4, 1), (64, 3, 1), (128, 1, 1), (64, 16, 2)])
def test_prompt_split_keys(dtype, dim, heads, kv):
    """Few queries at the end of long keys, whose keys are worked on in parts; next to
    sequences with hardly any keys, or none, of which some parts see nothing."""
    nq, nk = [3, 70, 1, 130, 5], [3000, 2600, 1, 2049, 2]
    check_prompt(*prompt_case(nq, nk, heads, kv, dim, dtype, heads), dtype)
    q, k, v, a, b = prompt_case([40, 0], [6000, 0], heads, kv, dim, dtype, heads + 1)
    first = check_prompt(q, k, v, a, b, dtype)
    for _ in range(3):
        again = G.grinqh_prompt_attention(q, k, v, a, b)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_prompt_long():
    check_prompt(*prompt_case([1500, 20], [1500, 2500], 2, 1, 128, "bf16", 7), "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_prompt_large_scores(dtype):
    """Scores of hundreds, whose running maximum rises many times."""
    q, k, v, a, b = prompt_case([400, 130], [400, 700], 2, 1, 128, dtype, 3)
    ramp = torch.linspace(0.2, 3, k.shape[0], device="cuda")[:, None, None]
    check_prompt(q * 3, (k * ramp).to(k.dtype), v, a, b, dtype, 0.3)


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_other_sequences_may_hold_nan(dim):
    """NaN and infinities in one sequence's q, k, v, and past the last one, reach no other."""
    q, k, v, a, b = prompt_case([50, 70, 200], [50, 70, 200], 4, 2, dim, "bf16", 13)
    q[50:120], k[50:120], v[50:120] = math.nan, math.inf, math.nan
    pad = torch.full((300, 2, dim), math.nan, dtype=k.dtype, device="cuda")
    check_prompt(q, torch.cat([k, pad]), torch.cat([v, pad]), a, b, "bf16", only=[0, 2])


def test_prompt_views_stream_and_graph():
    n = [200, 33, 128]
    fused = rand((361, 8, 128), "bf16", 3)
    q, k, v = fused.split([4, 2, 2], 1)
    cu = torch.tensor([0, 200, 233, 361], dtype=torch.int32).cuda()
    want = check_prompt(q.contiguous(), k.contiguous(), v.contiguous(), cu, cu, "bf16")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = G.grinqh_prompt_attention(q, k, v, cu, cu)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = G.grinqh_prompt_attention(q, k, v, cu, cu)
    for _ in range(3):
        kept[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept[0], want[0]) and torch.equal(kept[1], want[1])
    odd = torch.zeros(361, 8, 129, dtype=torch.bfloat16, device="cuda")  # rows that are not 16-byte aligned
    odd[..., 1:] = fused
    got = G.grinqh_prompt_attention(*odd[..., 1:].split([4, 2, 2], 1), cu, cu)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_prompt_rows_outside_sequences_are_not_written():
    q, k, v, a, b = prompt_case([40, 90], [40, 90], 2, 1, 128, "bf16", 17)
    cu = torch.tensor([10, 40, 100], dtype=torch.int32).cuda()
    out, lse = G.grinqh_prompt_attention(q, k, v, cu, cu)
    again = check_prompt(q[10:100].contiguous(), k[10:100].contiguous(), v[10:100].contiguous(), cu - 10, cu - 10, "bf16")
    assert torch.equal(out[10:100], again[0]) and torch.equal(lse[10:100], again[1])


def test_chunk_over_a_prefix_read_back():
    """The last tokens over the cache itself, and the same as a chunk over K and V read back from it."""
    kv, heads, dim, group = 2, 8, 128, 64
    case = cache_case("bf16", dim, group, kv, [230], 32, 61)
    cache, tables = case[:2]
    t = torch.arange(230).cuda()
    k, v = G.grinqh_kv4_gather(cache, tables[0].long()[t // 32] * 32 + t % 32, group)
    q = rand((1, 4, heads, dim), "bf16", 71)
    check_cached(q, case, group, "bf16")
    check_prompt(q[0], k, v, torch.tensor([0, 4], dtype=torch.int32).cuda(),
                 torch.tensor([0, 230], dtype=torch.int32).cuda(), "bf16")


# ------------------------------------------------------------------ refusals
def test_refusals():
    cache = G.grinqh_kv4_cache(4, 2, 128, 16, 128)
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(3).cuda()
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device="cuda")
    tables = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 3], dtype=torch.int32).cuda()
    calls = [
        lambda: G.grinqh_kv4_append(k.float(), k.float(), cache, slots),
        lambda: G.grinqh_kv4_append(k, k.half(), cache, slots),
        lambda: G.grinqh_kv4_append(k[:, :1], k[:, :1], cache, slots),
        lambda: G.grinqh_kv4_append(k[..., :64], k[..., :64], cache, slots),
        lambda: G.grinqh_kv4_append(k, k, cache, slots.int()),
        lambda: G.grinqh_kv4_append(k, k, cache, slots[:2]),
        lambda: G.grinqh_kv4_append(k, k, cache, slots.cpu()),
        lambda: G.grinqh_kv4_append(k, k, cache, slots, 64),
        lambda: G.grinqh_kv4_append(k, k, cache, slots, 16),
        lambda: G.grinqh_kv4_append(k, k, cache.float(), slots),
        lambda: G.grinqh_kv4_append(k, k, cache[..., :-1], slots),
        lambda: G.grinqh_kv4_gather(cache, slots, 128, torch.float32),
        lambda: G.grinqh_kv4_gather(cache.cpu(), slots.cpu(), 128),
        lambda: G.grinqh_kv4_attention(q[..., :64], cache, tables, lens),
        lambda: G.grinqh_kv4_attention(q[:, :3], cache, tables, lens),
        lambda: G.grinqh_kv4_attention(q.float(), cache, tables, lens),
        lambda: G.grinqh_kv4_attention(q, cache, tables.long(), lens),
        lambda: G.grinqh_kv4_attention(q, cache, tables, lens.long()),
        lambda: G.grinqh_kv4_attention(q, cache, tables, lens.repeat(2)),
        lambda: G.grinqh_kv4_attention(q.expand(1, 9, 8, 128), cache, tables, lens),
        lambda: G.grinqh_kv4_attention(q, cache, tables, lens, 128, -1.0),
        lambda: G.grinqh_kv4_attention(q, cache, tables, lens, 128, math.nan),
        lambda: G.grinqh_prompt_attention(k, k, k, cu, cu, 0.0),
        lambda: G.grinqh_prompt_attention(k, k, k, cu, cu, math.inf),
        lambda: G.grinqh_prompt_attention(k, k.half(), k.half(), cu, cu),
        lambda: G.grinqh_prompt_attention(k[:, :1], k, k, cu, cu),
        lambda: G.grinqh_prompt_attention(k, k, k[:2], cu, cu),
        lambda: G.grinqh_prompt_attention(k, k, k, cu.long(), cu),
        lambda: G.grinqh_prompt_attention(k, k, k, cu, cu[:1]),
        lambda: G.grinqh_prompt_attention(k[..., :32], k[..., :32], k[..., :32], cu, cu),
        lambda: G.grinqh_prompt_attention(k.cpu(), k.cpu(), k.cpu(), cu, cu),
    ]
    for i, call in enumerate(calls):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
            pytest.fail(f"call {i} was accepted")
    for bad in ((128, 16, 48), (128, 10, 64), (64, 16, 128), (96, 16, 32)):
        with pytest.raises(ValueError):
            G.grinqh_kv4_cache(4, 2, bad[0], bad[1], bad[2])


def test_nothing_to_do():
    cache = G.grinqh_kv4_cache(1, 2, 128, 16, 128)
    none = torch.zeros(0, 2, 128, dtype=torch.bfloat16, device="cuda")
    G.grinqh_kv4_append(none, none, cache, torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert not cache.any()
    k, v = G.grinqh_kv4_gather(cache, torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert k.shape == v.shape == (0, 2, 128)
    out, lse = G.grinqh_kv4_attention(none, cache, torch.zeros(0, 1, dtype=torch.int32, device="cuda"),
                                      torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 2, 128) and lse.shape == (0, 2)
    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = G.grinqh_prompt_attention(none, none, none, cu, cu)
    assert out.shape == (0, 2, 128) and lse.shape == (0, 2)
