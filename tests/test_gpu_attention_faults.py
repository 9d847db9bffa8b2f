"""What a reading of the attention operators and of what they share with the linears found
wrong, each held by a test: workspaces of captured graphs,
caches without heads, expanded inputs, joins of many sequences in a CTA, a block
that is full, waits that are lost, values of V
of very different size.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from oracle import attention as A  # noqa: E402

from grinqh import attention as G  # noqa: E402
from grinqh.kernel import grinqh_gemm_or_gemv  # noqa: E402
from grinqh.utils import pack_codes  # noqa: E402


@pytest.fixture(autouse=True)
def no_wait_is_lost():
    G.grinqh_check_waits()
    yield
    G.grinqh_check_waits()


def rand(shape, seed, dtype=torch.bfloat16, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[-1:], generator=g))
    return x.to(dtype).cuda()


def filled_cache(lens, kv, dim, group, page, seed, dtype=torch.bfloat16):
    """A cache with the sequences' random K and V, its tables and lengths."""
    need = [-(-n // page) for n in lens]
    cache = G.grinqh_kv4_cache(sum(need) + 1, kv, dim, page, group)
    order = np.random.default_rng(seed).permutation(sum(need) + 1)
    tables, at = np.zeros((len(lens), max(need)), np.int32), 0
    for b, n in enumerate(lens):
        tables[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        t = np.arange(n)
        slots = torch.from_numpy(tables[b, t // page].astype(np.int64) * page + t % page).cuda()
        G.grinqh_kv4_append(rand((n, kv, dim), seed + 2 * b, dtype), rand((n, kv, dim), seed + 2 * b + 1, dtype),
                            cache, slots, group)
    return cache, torch.from_numpy(tables).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


# ------------------------------------------------------------------ workspaces of captured graphs
def small_and_large(kind):
    """A call with a workspace, and one on a larger workspace."""
    if kind == "cached":
        cache, tables, lens = filled_cache([4000, 9, 1200], 2, 128, 64, 64, 1)
        few, many = rand((3, 8, 128), 2), rand((3, 4, 8, 128), 3)  # 4 query rows a kv head, and 16
        return (lambda: G.grinqh_kv4_attention(few, cache, tables, lens, 64),
                lambda: G.grinqh_kv4_attention(many, cache, tables, lens, 64))
    if kind == "prompt":  # keys in 4 parts, and in 2 parts of four times the items
        cu = [torch.tensor([0, n], dtype=torch.int32).cuda() for n in (40, 160, 6000)]
        k, v = rand((6000, 8, 128), 4), rand((6000, 8, 128), 5)
        few, many = rand((40, 32, 128), 6), rand((160, 32, 128), 7)
        return (lambda: G.grinqh_prompt_attention(few, k, v, cu[0], cu[2]),
                lambda: G.grinqh_prompt_attention(many, k, v, cu[1], cu[2]))
    g = torch.Generator(device="cuda").manual_seed(3)
    w = pack_codes(torch.randint(-128, 128, (4096, 4096), dtype=torch.int8, device="cuda", generator=g), 8)
    s = torch.full((32, 4096), 0.01, dtype=torch.bfloat16, device="cuda")
    few, many = rand((16, 4096), 8), rand((512, 4096), 9)
    return (lambda: (grinqh_gemm_or_gemv(few, w, s, None, 8, 128, 1024, [0.0] * 4),),
            lambda: (grinqh_gemm_or_gemv(many, w, s, None, 8, 128, 1024, [0.0] * 4),))


def graph_of(call, stream):
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        kept = call()
    return graph, kept


@pytest.mark.parametrize("kind", ["cached", "prompt", "linear"])
def test_graph_outlives_its_streams_workspace(kind):
    """A graph captured on a stream that has a workspace is replayed after a call on that
    stream has had it replaced by a larger one and its memory has been given to tensors."""
    few, many = small_and_large(kind)
    stream = torch.cuda.Stream(priority=-1)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        want = [x.clone() for x in few()]
    graph, kept = graph_of(few, stream)
    with torch.cuda.stream(stream):
        many()
        others = [torch.full((n,), 0xA5, dtype=torch.uint8, device="cuda") for n in (1 << 20, 8 << 20, 10 << 20) for _ in range(6)]
    torch.cuda.synchronize()
    for _ in range(3):
        for x in kept:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(kept, want))
    assert all(bool((x == 0xA5).all()) for x in others)


@pytest.mark.parametrize("kind", ["cached", "prompt", "linear"])
def test_graph_replays_beside_calls_on_its_stream(kind):
    """A replay on one stream and calls on the stream that it was captured on, at one time."""
    few, _ = small_and_large(kind)
    stream, other = torch.cuda.Stream(priority=-1), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        want = [x.clone() for x in few()]
    graph, kept = graph_of(few, stream)
    outs = []
    for _ in range(30):
        with torch.cuda.stream(other):
            graph.replay()
            outs.append([x.clone() for x in kept])
        with torch.cuda.stream(stream):
            outs.append(few())
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for out in outs for x, y in zip(out, want))


def test_graph_of_several_calls():
    """Calls of different sizes in one capture, the larger ones behind the smaller."""
    pairs = [small_and_large(kind) for kind in ("linear", "cached", "prompt")]
    calls = [call for pair in pairs for call in pair]
    want = [[x.clone() for x in call()] for call in calls]
    graph, kept = graph_of(lambda: [call() for call in calls + calls], torch.cuda.Stream())
    for _ in range(3):
        for out in kept:
            for x in out:
                x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for out, ref in zip(kept, want + want):
            assert all(torch.equal(x, y) for x, y in zip(out, ref))


# ------------------------------------------------------------------ refusals
def test_cache_without_heads_is_refused():
    cache = G.grinqh_kv4_cache(4, 0, 128, 16, 128)
    none = torch.zeros(3, 0, 128, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device="cuda")
    tables, lens = torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError):
        G.grinqh_kv4_attention(q, cache, tables, lens)
    with pytest.raises(RuntimeError):
        G.grinqh_kv4_attention(q[:, :0], cache, tables, lens)
    with pytest.raises(RuntimeError):
        G.grinqh_kv4_append(none, none, cache, torch.arange(3).cuda())
    with pytest.raises(RuntimeError):
        G.grinqh_prompt_attention(q, none[:1], none[:1], lens, lens)


# ------------------------------------------------------------------ strides
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_of_expanded_and_transposed_inputs(dim):
    """K and V of one head expanded over the kv heads, of one token over all; and q, k, v
    held head by head."""
    cu = torch.tensor([0, 70, 203], dtype=torch.int32).cuda()
    q, k, v = rand((203, 8, dim), 1), rand((203, 4, dim), 2), rand((203, 4, dim), 3)

    def same(q, k, v):
        got = G.grinqh_prompt_attention(q, k, v, cu, cu)
        want = G.grinqh_prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, cu)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

    same(q, k[:, :1].expand(-1, 4, -1), v[:, :1].expand(-1, 4, -1))
    same(q[:1].expand(203, -1, -1), k[:1].expand(203, -1, -1), v)
    same(q[:, :1].expand(-1, 8, -1), k, v)
    same(*(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)))


def test_cache_of_expanded_inputs():
    one, tokens = rand((40, 1, 128), 1), rand((1, 4, 128), 2)
    slots = torch.arange(40).cuda()
    caches = [G.grinqh_kv4_cache(3, 4, 128, 16, 64) for _ in range(2)]
    G.grinqh_kv4_append(one.expand(-1, 4, -1), tokens.expand(40, -1, -1), caches[0], slots, 64)
    G.grinqh_kv4_append(one.expand(-1, 4, -1).contiguous(), tokens.expand(40, -1, -1).contiguous(), caches[1], slots, 64)
    assert torch.equal(*caches)
    tables, lens = torch.arange(3, dtype=torch.int32).cuda()[None].expand(2, -1), torch.tensor([40, 17]).int().cuda()
    q = rand((2, 1, 128), 3).expand(-1, 8, -1)
    got = G.grinqh_kv4_attention(q, caches[0], tables, lens, 64)
    want = G.grinqh_kv4_attention(q.contiguous(), caches[0], tables.contiguous(), lens, 64)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------ joins
@pytest.mark.parametrize("dim,group", [(128, 32), (128, 64), (64, 32)])
def test_cached_attention_of_many_short_sequences(dim, group):
    """Every CTA holds many sequences and heads that several of its warps share: each is what
    the sequence gives alone, up to the order of fp32 sums."""
    lens = [37 + 11 * (i % 23) for i in range(400)]
    cache, tables, start = filled_cache(lens, 2, dim, group, 32, 5)
    q = rand((400, 8, dim), 6)
    out, lse = G.grinqh_kv4_attention(q, cache, tables, start, group)
    for _ in range(3):
        again = G.grinqh_kv4_attention(q, cache, tables, start, group)
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    for b in list(range(0, 400, 37)) + [399]:
        one = G.grinqh_kv4_attention(q[b:b + 1], cache, tables[b:b + 1], start[b:b + 1], group)
        # weights in 11 bits and one rounding to bf16 on each side; codes x scale reach 3 x the values, 5 sigma
        assert (out[b:b + 1] - one[0]).abs().max() <= 2 * (2.0**-11 * 15 + 2.0**-8 * one[0].abs().max())
        assert (lse[b:b + 1] - one[1]).abs().max() <= 1e-5 * (1 + one[1].abs().max())


# ------------------------------------------------------------------ the block
def test_block_refuses_tokens_behind_its_pages():
    """One page of 16 tokens a sequence: what does not fit is refused on the host, and leaves
    the block as it was."""
    from grinqh.attention_block import AttentionBlock
    block = AttentionBlock(2, 10, hidden=512, heads=4, kv_heads=2, head_dim=64, page=16, group=32)
    rows = lambda n: rand((n, 512), n)  # noqa: E731
    for bad in (0, 3, 34):
        with pytest.raises(ValueError):
            block.prompt(rows(bad))
    block.prompt(rows(30))
    cache = block.cache.clone()
    for call, n in ((block.prompt, 4), (block.token, 4), (block.token, 1)):
        with pytest.raises(ValueError):
            call(rows(n))
    assert block.length == 15 and torch.equal(block.cache, cache)
    block.token(rows(2))
    for call in (block.token, block.prompt):
        with pytest.raises(ValueError):
            call(rows(2))
    assert block.length == 16 and block.lens.tolist() == [16, 16]


# ------------------------------------------------------------------ waits
def lost_rows(call, want, monkeypatch):
    """Runs `call` with every wait lost, `want` being what it returns without: rows that need
    nothing are right and all others NaN, the loss is reported once, and later calls are right."""
    monkeypatch.setenv("GRINQH_ATTENTION_WAIT_US", "0")
    outs = [call() for _ in range(3)]
    torch.cuda.synchronize()
    monkeypatch.delenv("GRINQH_ATTENTION_WAIT_US")
    again = call()  # the flag of the lost calls is still up
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    with pytest.raises(RuntimeError, match="gave up"):
        G.grinqh_check_waits()
    G.grinqh_check_waits()
    for out, lse in outs:
        gone = lse.isnan()
        assert torch.equal(gone, out.isnan().all(-1)) and torch.equal(gone, out.isnan().any(-1))
        assert torch.equal(out[~gone], want[0][~gone]) and torch.equal(lse[~gone], want[1][~gone])
        assert gone[~want[1].isneginf()].all()


@pytest.mark.parametrize("lens,dim,group,new", [([20000, 3, 9000], 128, 64, 1), ([700] * 40, 128, 32, 1), ([50, 0, 31], 64, 32, 4),
                                                ([5000, 800], 128, 128, 4)])
def test_cached_attention_waits_are_bounded(lens, dim, group, new, monkeypatch):
    cache, tables, seq = filled_cache(lens, 2, dim, group, 64, 11)
    q = rand((len(lens), new, 8, dim), 12)
    call = lambda: G.grinqh_kv4_attention(q, cache, tables, seq, group)  # noqa: E731
    lost_rows(call, call(), monkeypatch)


def test_check_of_waits_is_not_captured():
    x = torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError):
            G.grinqh_check_waits()


@pytest.mark.parametrize("nq,nk,heads,kv,dim", [([1500], [1500], 2, 1, 128), ([600] * 40, [900] * 40, 8, 2, 64), ([30], [9000], 8, 2, 128),
                                                ([20, 700, 5], [5000, 700, 0], 4, 2, 64)])
def test_prompt_attention_waits_are_bounded(nq, nk, heads, kv, dim, monkeypatch):
    cu = [torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32).cuda() for n in (nq, nk)]
    q, k, v = rand((sum(nq), heads, dim), 1), rand((sum(nk), kv, dim), 2), rand((sum(nk), kv, dim), 3)
    call = lambda: G.grinqh_prompt_attention(q, k, v, *cu)  # noqa: E731
    lost_rows(call, call(), monkeypatch)


# ------------------------------------------------------------------ range
def one_sequence(k, v, group, page=16):
    """A cache of k and v [n, 1, D], tables and lengths, and what it holds in 64 bits."""
    n = k.shape[0]
    pages = -(-n // page)
    cache = G.grinqh_kv4_cache(pages, 1, k.shape[2], page, group)
    G.grinqh_kv4_append(k, v, cache, torch.arange(n).cuda(), group)
    held = A.read_tokens(cache.cpu().numpy().reshape(-1, cache.shape[3]), k.shape[2], group, "bf16")
    tables = torch.arange(pages, dtype=torch.int32).cuda()[None]
    return cache, tables, torch.tensor([n], dtype=torch.int32).cuda(), [x[:n, None] for x in held]


def scales_of(v, group):
    g = v.reshape(*v.shape[:-1], -1, group)
    return ((g.max(-1, keepdims=True) - g.min(-1, keepdims=True)) / 15 * np.ones(group)).reshape(v.shape)


@pytest.mark.parametrize("what", ["group", "token"])
@pytest.mark.parametrize("power", [12, 20, 24])
@pytest.mark.parametrize("dim,group,heads", [(128, 64, 4), (64, 32, 12), (128, 32, 1)])
def test_cached_attention_of_values_of_very_different_size(what, power, dim, group, heads):
    """One group of V, or one token that hardly counts, is 2^power larger than the rest. A weight
    is off by 2^-11 of itself (twice: its own rounding and the scale's product) and, in f16's smallest
    step, by 2^-35 of the row's largest times the largest scale over its own; a code is at most 15."""
    n = 300
    k, v, q = rand((n, 1, dim), 1), rand((n, 1, dim), 2), rand((1, heads, dim), 3)
    big = 2.0**power
    if what == "group":
        v[:, :, :group] *= big
    else:
        q = q.abs()
        k[7], v[7] = -3.0, v[7] * big
    cache, tables, lens, (kr, vr) = one_sequence(k, v, group)
    out, lse = G.grinqh_kv4_attention(q, cache, tables, lens, group)
    x = q.double().cpu().numpy()
    ref, ref_lse, _, reach = A.attention(x, kr, vr, dim**-0.5)
    s = scales_of(vr, group)
    size = A.attention(x, kr, np.abs(vr) + 15 * s, dim**-0.5)[2]
    top = (x[0] @ kr[:, 0].T).max(-1) * dim**-0.5
    share = np.exp(top - ref_lse[0])[None, :, None]  # of the row's largest weight
    d = 2.0**-20 * (3 * reach.max() + 1)
    off = np.abs(out.double().cpu().numpy() - ref)
    limit = (2.0**-10 + 2 * d) * size + 2.0**-8 * np.abs(ref) + n * share * 15 * 2.0**-35 * s.max() + 2.0**-20 * size
    assert (off <= limit).all(), f"worst {np.max(off / limit)} of the bound"


@pytest.mark.parametrize("q_power,k_power,v_power", [(0, 0, 118), (0, 0, -110), (117, -119, 0), (-100, 100, 0)])
def test_cached_attention_of_huge_and_tiny_values(q_power, k_power, v_power):
    """Values near the ends of bf16's range, with scores and outputs within it."""
    n = 100
    k, v, q = rand((n, 1, 128), 1) * 2.0**k_power, rand((n, 1, 128), 2).clamp(-3, 3), rand((1, 4, 128), 3) * 2.0**q_power
    cache, tables, lens, (kr, vr) = one_sequence(k, v * 2.0**v_power, 128)
    out, lse = G.grinqh_kv4_attention(q, cache, tables, lens, 128)
    ref, ref_lse, _, _ = A.attention(q.double().cpu().numpy(), kr, vr, 128**-0.5)
    # weights in 11 bits times codes up to 3 |v|, out rounded to 8; a score's products near 2^-126 lose bits: 1 %
    size = np.abs(vr).max()
    assert np.abs(out.double().cpu().numpy() - ref).max() <= 0.01 * size
    assert np.abs(lse.double().cpu().numpy() - ref_lse).max() <= 0.01 * (1 + np.abs(ref_lse).max())
