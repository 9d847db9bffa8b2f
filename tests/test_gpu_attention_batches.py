"""Prompt attention on batches with more items of work than a B200 has SMs, more than 32
sequences and many query heads per kv head, against the numpy oracle.

Tolerances as in the operators' other tests, derived before any run: weights enter the
products in the inputs' type (unit roundoff 2^-8 or 2^-11), scores are off by a few units of 2^-22 of
their largest sum, which moves a weight by that factor, and out is rounded once.
"""
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


@pytest.fixture(autouse=True)
def no_wait_is_lost():
    yield
    G.grinqh_check_waits()


def rand(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(DT[dtype])


def check(nq, nk, heads, kv, dim, dtype, only, seed=0):
    a, b = (np.concatenate([[0], np.cumsum(n)]) for n in (nq, nk))
    cu_q, cu_k = (torch.tensor(x, dtype=torch.int32).cuda() for x in (a, b))
    q, k, v = rand((a[-1], heads, dim), dtype, seed + 1), rand((b[-1], kv, dim), dtype, seed + 2), rand((b[-1], kv, dim), dtype, seed + 3)
    out, lse = G.grinqh_prompt_attention(q, k, v, cu_q, cu_k)
    for _ in range(3):
        again = G.grinqh_prompt_attention(q, k, v, cu_q, cu_k)
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    seen = np.repeat(np.array(nk) - np.array(nq), nq) + np.concatenate([np.arange(n) for n in nq]) + 1
    none = torch.from_numpy(seen <= 0).cuda()
    assert torch.equal(lse.isneginf().all(-1), none) and torch.equal(lse.isneginf().any(-1), none)
    assert not out[none].any() and not out.isnan().any() and not lse.isnan().any()
    for i in only:
        x, y, z = (t.double().cpu().numpy() for t in (q[a[i]:a[i + 1]], k[b[i]:b[i + 1]], v[b[i]:b[i + 1]]))
        ref, ref_lse, size, reach = A.attention(x, y, z, dim**-0.5)
        d = 2.0**-20 * (reach[..., None] + 1)
        limit = (UNIT[dtype] + 2 * d) * size + UNIT[dtype] * np.abs(ref) + nk[i] * 2.0**-24 * size.max(initial=0) + 1e-30
        off = np.abs(out[a[i]:a[i + 1]].double().cpu().numpy() - ref)
        assert (off <= limit).all(), f"sequence {i}: worst {np.max(off / limit)} of the bound"
        there = ~np.isneginf(ref_lse)
        off = np.abs(lse[a[i]:a[i + 1]].double().cpu().numpy()[there] - ref_lse[there])
        assert (off <= 2.0**-20 * (reach + 1 + np.abs(ref_lse))[there]).all()


def ragged(count, most, seed, prefix=0):
    """Lengths in 1..most, with sequences that have no queries, no keys, or more queries than keys
    among them, also next to a border of 32."""
    rng = np.random.default_rng(seed)
    nq = rng.integers(1, most + 1, count)
    nk = nq + (rng.integers(0, prefix + 1, count) if prefix else 0)
    for i, (x, y) in enumerate(((0, 40), (70, 0), (90, 33), (0, 0))):
        for at in (i + 2, count // 2 + i, 29 + i, 32 + i, count - 5 + i):
            if at < count:
                nq[at], nk[at] = x, y
    return nq.tolist(), nk.tolist()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("count,most,heads,kv", [(20, 700, 16, 4), (31, 300, 8, 8), (32, 150, 32, 8), (33, 200, 24, 8),
                                                 (70, 260, 8, 2), (100, 30, 16, 8)])
def test_batches_of_many_items(dtype, dim, count, most, heads, kv):
    """Several items a CTA, taken over from CTAs that have not started; sequences found among
    up to 32 held in registers, and among more."""
    nq, nk = ragged(count, most, count)
    check(nq, nk, heads, kv, dim, dtype, [0, 3, 4, 12, count // 2 + 2, count - 6, count - 1])


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64)])
def test_batches_of_many_items_after_prefixes(dtype, dim):
    nq, nk = ragged(40, 200, 3, 1500)
    check(nq, nk, 12, 4, dim, dtype, [0, 4, 7, 22, 31, 34, 39])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("count,kv", [(33, 1), (66, 1)])
def test_split_keys_of_many_sequences(dim, count, kv):
    """A query or two of each of many long sequences: their keys in parts, joined."""
    rng = np.random.default_rng(count)
    nq = [1] * count
    nk = rng.integers(700, 2000, count)
    nk[3], nk[32] = 0, 1
    nq[31 % count], nq[20] = 2, 0
    check(nq, nk.tolist(), 4 * kv, kv, dim, "bf16", [0, 3, 20, 31, 32, count - 1])


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("bf16", 64)])
@pytest.mark.parametrize("group", [5, 8, 16, 33, 64, 100, 128])
def test_many_heads_per_kv_head(dtype, dim, group):
    """Tiles of 25 tokens down to one, some with rows that no head fills."""
    check([70, 1, 3], [70, 200, 2], 2 * group, 2, dim, dtype, [0, 1, 2], group)
    check([9], [1300], group, 1, dim, dtype, [0], group)
