"""The dense model over the 8-bit cache: its operators run together."""

import pytest
import torch
import torch.nn.functional as F

from cxlsparse_b200 import ops
from cxlsparse_b200.dense import DenseCacheModel
from cxlsparse_b200.model import NSAConfig, rms_norm, rotary

pytestmark = pytest.mark.gpu

CFG = dict(layers=2, hidden=256, q_heads=8, kv_heads=2, ffn=512, vocab=500)


def plain(model, history):
    """Logits of one user's tokens with 16-bit keys and values, in fp32."""
    cfg = model.cfg
    f = 1.0 / (cfg.rope_theta ** (torch.arange(0, 64, 2, device="cuda").float() / 64))
    hidden = model.embed[history].float()
    n, positions = len(history), torch.arange(len(history), device="cuda")
    mask = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    for w in model.layers:
        w = {k: t.float() for k, t in w.items()}
        x = rms_norm(hidden, w["in_norm"], cfg.rms_eps)
        q, k, v = F.linear(x, w["qkv"]).view(n, -1, 64).split([8, 2, 2], 1)
        q, k = rotary(q, k, positions, f)
        k, v = (t.repeat_interleave(4, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) / 8
        p = s.masked_fill(~mask, float("-inf")).softmax(-1)
        hidden = hidden + F.linear(torch.einsum("hqk,khd->qhd", p, v).flatten(1), w["o"])
        x = rms_norm(hidden, w["post_norm"], cfg.rms_eps)
        gate, up = F.linear(x, w["gate_up"]).chunk(2, -1)
        hidden = hidden + F.linear(F.silu(gate) * up, w["down"])
    return F.linear(rms_norm(hidden, model.norm.float(), cfg.rms_eps), model.embed.float())


@pytest.mark.parametrize("format,page_size", [("e4m3", 64), ("int8", 16)])
def test_prefill_suffix_and_decode_follow_the_plain_model(cuda, format, page_size):
    """Ragged prefill, a suffix of some users, single tokens of others. The
    cache's codes carry at most 4 (e4m3) or about 7 bits, in two layers of
    attention whose output is a small part of the hidden state (weights 0.02):
    logits within 5 percent of their norm, and the argmax's logit close."""
    model = DenseCacheModel(NSAConfig(**CFG), users=3, max_tokens=400, page_size=page_size,
                            format=format)
    g = torch.Generator(device="cuda").manual_seed(0)
    history = [torch.randint(0, 500, (n,), generator=g, device="cuda") for n in (331, 70, 12)]
    steps = [(300, 64, 0), (0, 1, 9), (30, 4, 1), (1, 1, 1), (0, 0, 1)]
    at = [0, 0, 0]
    for counts in steps:
        tokens = torch.cat([history[b][at[b]:at[b] + n] for b, n in enumerate(counts)])
        logits = model.step(tokens, list(counts))
        at = [a + n for a, n in zip(at, counts)]
        row = 0
        for b, n in enumerate(counts):
            if n:
                want = plain(model, history[b][:at[b]])[-n:]
                got = logits[row:row + n].float()
                assert (got - want).norm() <= 0.05 * want.norm()
            row += n
    assert at == [331, 70, 12] == model.lengths
    model.check()
    # Records read back feed the block summaries.
    records = model.records(1, 0, 64, 256)
    assert records.shape == (256, 2, 128) and records.dtype == torch.bfloat16
    summaries = ops.block_summaries(records, 64)
    torch.testing.assert_close(summaries.float(), records.float().view(4, 64, 2, 128).mean(1),
                               rtol=2 ** -7, atol=1e-3)
    with pytest.raises(ValueError):
        model.step(history[0], [331, 0, 0])
    with pytest.raises(ValueError):
        model.records(0, 1, 60, 20)
