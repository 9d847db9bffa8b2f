"""The numpy oracle of the 4-bit cache: layout and quantization against their definitions (CPU)."""
import numpy as np
import pytest

from oracle import attention as A

SHAPES = [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)]


@pytest.mark.parametrize("dim,group", SHAPES)
def test_record_holds_every_channel_once(dim, group):
    """Writing 16 tokens fills every byte of a record exactly, and reading gives them back."""
    rng = np.random.default_rng(dim + group)
    x = A.to_bits(rng.standard_normal((2, 16, dim)).astype(np.float32), "bf16")
    rec = np.full((1, A.record_bytes(dim, group)), 0xA5, np.uint8)
    parts = [A.quantize(y, "bf16", group) for y in x]
    for t in rng.permutation(16):
        A.write_token(rec[0], t, group, *[tuple(z[t] for z in p) for p in parts])
    for got, (u, s, z) in zip(A.read_tokens(rec, dim, group, "bf16"), parts):
        sc, zr = A.to_f32(s, "bf16").astype(np.float64), A.to_f32(z, "bf16").astype(np.float64)
        want = u.reshape(16, -1, group) * sc[..., None] + zr[..., None]
        assert np.array_equal(got, want.reshape(16, dim))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim,group", SHAPES)
def test_quantization_is_within_half_a_step(dim, group, dtype):
    """|value - x| <= scale / 2, plus what rounding the scale moves the top code: 15 scale u."""
    rng = np.random.default_rng(7)
    x = A.to_bits((rng.standard_normal((40, dim)) * np.exp(rng.standard_normal((40, 1)))).astype(np.float32), dtype)
    u, s, z = A.quantize(x, dtype, group)
    sc, zr = A.to_f32(s, dtype).astype(np.float64), A.to_f32(z, dtype).astype(np.float64)
    value = u.reshape(40, -1, group) * sc[..., None] + zr[..., None]
    unit = 2.0**-8 if dtype == "bf16" else 2.0**-11
    off = np.abs(value - A.to_f32(x, dtype).astype(np.float64).reshape(value.shape))
    assert (off <= sc[..., None] * (0.5 + 15 * unit + 1e-5)).all()


def test_constant_group_is_exact():
    x = A.to_bits(np.full((1, 128), -3.25, np.float32), "bf16")
    u, s, z = A.quantize(x, "bf16", 64)
    assert not u.any() and not s.any() and (A.to_f32(z, "bf16") == -3.25).all()


def test_rows_without_keys():
    q = np.ones((3, 2, 4))
    out, lse, _, _ = A.attention(q, np.ones((1, 1, 4)), np.full((1, 1, 4), 2.0), 0.5)
    assert not out[:2].any() and np.isneginf(lse[:2]).all()
    assert np.allclose(out[2], 2.0) and np.allclose(lse[2], 2.0)
