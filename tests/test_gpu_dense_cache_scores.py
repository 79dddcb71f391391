"""The dense model over the 8-bit cache with attention that matters."""

import pytest
import torch
import torch.nn.functional as F

from cxlsparse_b200.dense import DenseCacheModel
from cxlsparse_b200.model import NSAConfig, rms_norm, rotary

pytestmark = pytest.mark.gpu

CFG = dict(layers=2, hidden=256, q_heads=8, kv_heads=2, ffn=512, vocab=500)


def plain(model, user, tokens, turn=True, flat=False):
    """Logits of a user's newest tokens in fp32, with the keys and values that the
    cache holds (so only the newest tokens pass through the layers). ``turn`` and
    ``flat`` leave the rotation out and make all scores 0: planted mistakes."""
    cfg, length = model.cfg, model.lengths[user]
    n = len(tokens)
    f = 1.0 / (cfg.rope_theta ** (torch.arange(0, 64, 2, device="cuda").float() / 64))
    positions = torch.arange(length - n, length, device="cuda")
    mask = torch.arange(length, device="cuda") <= positions[:, None]
    table = torch.tensor([model.pages[user]], dtype=torch.int32, device="cuda")
    zero, ends = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0], [0, length]))
    hidden = model.embed[tokens].float()
    for w, cache in zip(model.layers, model.caches):
        w = {name: t.float() for name, t in w.items()}
        x = rms_norm(hidden, w["in_norm"], cfg.rms_eps)
        q = F.linear(x, w["qkv"]).view(n, -1, 64)[:, :8]
        if turn:
            q, _ = rotary(q, q, positions, f)
        k, v = (t.repeat_interleave(4, 1) for t in cache.read(table, zero, ends, total=length,
                                                              dtype=torch.float32))
        s = torch.einsum("qhd,khd->hqk", q, k) / 8 * (0.0 if flat else 1.0)
        p = s.masked_fill(~mask, float("-inf")).softmax(-1)
        hidden = hidden + F.linear(torch.einsum("hqk,khd->qhd", p, v).flatten(1), w["o"])
        x = rms_norm(hidden, w["post_norm"], cfg.rms_eps)
        gate, up = F.linear(x, w["gate_up"]).chunk(2, -1)
        hidden = hidden + F.linear(F.silu(gate) * up, w["down"])
    return F.linear(rms_norm(hidden, model.norm.float(), cfg.rms_eps), model.embed.float())


@pytest.mark.parametrize("format,page_size", [("e4m3", 64), ("int8", 16)])
def test_steps_follow_the_plain_model_over_the_same_cache(cuda, format, page_size):
    """Scores of spread about 2.5 and an output projection five times as large.
    Against fp32 the model rounds to bf16 (2^-9) about a dozen times a layer, and
    its scores by about 2.5 * 2^-8: logits within 3 percent of their norm, and
    the largest one within 5 percent. A model without the rotation, or with flat
    scores, is off by several times that."""
    model = DenseCacheModel(NSAConfig(**CFG), users=3, max_tokens=400, page_size=page_size,
                            format=format)
    for w in model.layers:
        w["qkv"][:10 * 64] *= 5
        w["o"] *= 5
    g = torch.Generator(device="cuda").manual_seed(0)
    history = [torch.randint(0, 500, (n,), generator=g, device="cuda") for n in (331, 70, 12)]
    at = [0, 0, 0]
    for counts in ((300, 64, 0), (0, 1, 9), (30, 4, 1), (1, 1, 1), (0, 0, 1)):
        new = [history[b][at[b]:at[b] + n] for b, n in enumerate(counts)]
        logits = model.step(torch.cat(new), list(counts)).float()
        at = [a + n for a, n in zip(at, counts)]
        row = 0
        for b, n in enumerate(counts):
            if not n:
                continue
            got, want = logits[row:row + n], plain(model, b, new[b])
            row += n
            assert (got - want).norm() <= 0.03 * want.norm()
            top, index = want.max(-1)
            assert ((got.gather(1, index[:, None])[:, 0] - top).abs() <= 0.05 * top).all()
            if at[b] > 60:
                for mistake in (dict(turn=False), dict(flat=True)):
                    assert (plain(model, b, new[b], **mistake) - want).norm() > 0.1 * want.norm()
    model.check()
