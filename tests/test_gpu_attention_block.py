"""The attention block on GRINQH linears and the 4-bit cache, its phases against each other."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from grinqh.attention_block import AttentionBlock, main  # noqa: E402
from oracle import attention as A  # noqa: E402


def test_phases_follow_one_another():
    """After a prompt, a chunk and two tokens, the last token's attention is that over the
    cache's contents, and those are the block's own K and V quantized."""
    seqs, shape = 3, dict(hidden=512, heads=8, kv_heads=2, head_dim=128, page=32, group=64)
    block = AttentionBlock(seqs, 100, **shape)
    kept, seen = [], {}
    append, project = block._append, block._project

    def keep(k, v, count):
        kept.append((k.reshape(seqs, count, 2, 128), v.reshape(seqs, count, 2, 128)))
        append(k, v, count)

    def note(x, count):
        seen["q"], k, v = project(x, count)
        return seen["q"], k, v

    block._append, block._project = keep, note
    block.o = lambda x: seen.setdefault("out", x) if x.shape[0] == seqs and block.length == 72 else x
    g = torch.Generator(device="cuda").manual_seed(5)
    rows = lambda n: torch.randn(n, 512, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    assert block.prompt(rows(seqs * 40)).shape == (seqs * 40, 1024)
    assert block.prompt(rows(seqs * 30)).shape == (seqs * 30, 1024)
    block.token(rows(seqs))
    block.token(rows(seqs))
    assert block.length == 72 and block.lens.tolist() == [72] * seqs
    host, tables = block.cache.cpu().numpy(), block.tables.cpu().numpy()
    for b in range(seqs):
        rec = host[tables[b]]
        k, v = (np.stack([A.read_tokens(rec[:, h].reshape(-1, rec.shape[-1]), 128, 64, "bf16")[i][:72]
                          for h in range(2)], 1) for i in (0, 1))
        for got, parts in ((k, [x[0][b] for x in kept]), (v, [x[1][b] for x in kept])):
            x = torch.cat(parts).contiguous()
            u, s, z = A.quantize(x.view(torch.int16).cpu().numpy().view(np.uint16), "bf16", 64)
            s, z = (A.to_f32(y, "bf16").astype(np.float64)[..., None] for y in (s, z))
            assert np.array_equal(got, (u.reshape(72, 2, 2, 64) * s + z).reshape(72, 2, 128))
        q = seen["q"].view(seqs, 1, 8, 128)[b].double().cpu().numpy()
        ref, _, size, reach = A.attention(q, k, v, 128**-0.5)
        out = seen["out"].view(seqs, 1, 8, 128)[b].double().cpu().numpy()
        # weights in 11 bits times codes up to 3 |v|, one rounding to bf16, scores to 2^-20
        limit = (3 * 2.0**-11 + 2.0**-19 * (reach[..., None] + 1)) * (size + np.abs(v).max()) + 2.0**-8 * np.abs(ref)
        assert (np.abs(out - ref) <= limit).all()


def test_command_runs(capsys):
    main(["--seqs", "2", "--prompt", "70", "--chunk", "33", "--gen", "3", "--page", "16", "--group", "64"])
    assert '"token_ms"' in capsys.readouterr().out
