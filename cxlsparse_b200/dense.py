"""A dense model over the 8-bit cache: whole histories in HBM, every token read.

The counterpart of the extend model for users whose history is kept in HBM:
the same layer (RMSNorm, q/k/v projections, o_proj, SwiGLU) with rotary
positions, ``QuantizedCache.append`` and dense ``QuantizedCache.attend`` in the
place of the selected-block transport and its three branches. One ``step``
takes any number of new tokens of any of the users (a prefill, a suffix, one
decoded token each); all layers share one page table. ``generate`` draws
several continuations of every user's history: candidates that share the
history's pages (``PageTable``), attend over it once for all
(``QuantizedCache.attend_shared``) and get their tokens from ``sample``, with
no host synchronisation between the steps. Weights are random N(0, 0.02) with a
fixed seed. No counterpart in the reference.

    python -m cxlsparse_b200.dense      # a prefill, decode steps, candidates, timed
"""

import torch
import torch.nn.functional as F

from .model import NSAConfig, rms_norm
from .pages import PageTable
from .quantized import QuantizedCache
from .rotary import Rotary
from .sampling import sample


class DenseCacheModel:
    """``candidates``: most continuations of each user that ``generate`` draws at
    once, of at most ``candidate_tokens`` tokens (their pages are kept ready)."""

    def __init__(self, cfg=None, *, users=1, max_tokens=4096, page_size=64, format="e4m3",
                 scaling=None, device="cuda", seed=0, candidates=0, candidate_tokens=64):
        self.cfg = cfg = cfg or NSAConfig()
        self.device = torch.device(device)
        g = torch.Generator(device="cpu").manual_seed(seed)

        def normal(*shape):
            return (torch.randn(*shape, generator=g) * 0.02).to(torch.bfloat16).to(self.device)

        d, q_dim, kv_dim = cfg.hidden, cfg.q_heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim
        self.embed = normal(cfg.vocab, d)
        ones = torch.ones(d, dtype=torch.bfloat16, device=self.device)
        self.norm = ones
        self.layers = [dict(in_norm=ones, post_norm=ones, qkv=normal(q_dim + 2 * kv_dim, d),
                            o=normal(d, q_dim), gate_up=normal(2 * cfg.ffn, d),
                            down=normal(d, cfg.ffn)) for _ in range(cfg.layers)]
        self.page_size, self.max_tokens = page_size, max_tokens
        width = -(-max_tokens // page_size)
        own = -(-(page_size - 1 + candidate_tokens) // page_size)  # pages of a candidate's own
        self.candidates, self.candidate_tokens = candidates, candidate_tokens
        self.caches = [QuantizedCache(users * (width + candidates * own), cfg.kv_heads,
                                      cfg.head_dim, page_size=page_size, format=format,
                                      device=self.device)
                       for _ in range(cfg.layers)]
        self.table = PageTable(self.caches, users * (1 + candidates), width + own) \
            if candidates else None
        self.rotary = Rotary(cfg.head_dim, theta=cfg.rope_theta, scaling=scaling,
                             device=self.device)
        # Pages are taken as tokens come, the last free one first; -1: none.
        self.free = list(range(users * width))
        self.pages = [[] for _ in range(users)]
        self.lengths = [0] * users

    def _tensor(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def _grow(self, counts):
        """Pages for counts[b] more tokens of each user; the step's
        (table, lengths, offsets, positions)."""
        for b, count in enumerate(counts):
            if count < 0 or self.lengths[b] + count > self.max_tokens:
                raise ValueError(f"user {b}: more than {self.max_tokens} tokens")
        positions, offsets = [], [0]
        for b, count in enumerate(counts):
            positions += range(self.lengths[b], self.lengths[b] + count)
            offsets.append(offsets[-1] + count)
            self.lengths[b] += count
            while len(self.pages[b]) * self.page_size < self.lengths[b]:
                self.pages[b].append(self.free.pop())
        width = max(1, max(len(p) for p in self.pages))
        table = self._tensor([p + [-1] * (width - len(p)) for p in self.pages])
        return table, self._tensor(self.lengths), self._tensor(offsets), self._tensor(positions)

    def step(self, tokens, counts):
        """Append ``counts[b]`` new tokens of each user (``tokens`` packed in
        user order) and return their logits [tokens, vocab]."""
        if len(tokens) != sum(counts) or len(counts) != len(self.lengths):
            raise ValueError("counts must cover the tokens, one entry a user")
        table, lengths, offsets, positions = self._grow(counts)
        most = max(counts)

        def attend(cache, q):
            return cache.attend(q, table, lengths, offsets, max_tokens=most)

        return self._forward(tokens, positions, (table, lengths, offsets), most, attend)

    def _forward(self, tokens, positions, rows, most, attend):
        """Logits of new tokens: appended at ``rows`` (table, lengths, offsets), of
        which no user has more than ``most``, then ``attend(cache, queries)``."""
        cfg = self.cfg
        hidden = self.embed[tokens]
        split = [cfg.q_heads * cfg.head_dim] + 2 * [cfg.kv_heads * cfg.head_dim]
        for w, cache in zip(self.layers, self.caches):
            x = rms_norm(hidden, w["in_norm"], cfg.rms_eps)
            q, k, v = (t.view(len(x), -1, cfg.head_dim)
                       for t in F.linear(x, w["qkv"]).split(split, -1))
            q, k = self.rotary.apply(q, k, positions)
            cache.append(k, v, *rows, max_tokens=most)
            mixed = attend(cache, q)
            hidden = hidden + F.linear(mixed.flatten(1), w["o"])
            x = rms_norm(hidden, w["post_norm"], cfg.rms_eps)
            gate, up = F.linear(x, w["gate_up"]).chunk(2, -1)
            hidden = hidden + F.linear(F.silu(gate) * up, w["down"])
        return F.linear(rms_norm(hidden, self.norm, cfg.rms_eps), self.embed)

    def generate(self, logits, uniforms, **settings):
        """Continuations of every user's history: tokens and their
        log-probabilities [users, candidates, steps], drawn (``sample``, with
        its settings, numbers or one for each user) from ``logits [users, vocab]`` after each history for the
        first token, and from the model for the others, with ``uniforms
        [users, candidates, steps]``. The histories stay as they are."""
        users = len(self.lengths)
        if uniforms.ndim != 3 or uniforms.shape[0] != users or len(logits) != users:
            raise ValueError("logits must be [users, vocab], uniforms [users, candidates, steps]")
        count, steps = uniforms.shape[1:]
        if not 1 <= count <= self.candidates or not 1 <= steps <= self.candidate_tokens:
            raise ValueError(f"at most {self.candidates} candidates of at most "
                             f"{self.candidate_tokens} tokens")
        pages, total = self.table, users * count
        rows = [p + [-1] * (pages.width - len(p)) for p in self.pages]
        rows += [[-1] * pages.width] * (pages.sequences - users)
        pages.adopt(self._tensor(rows),
                    self._tensor(self.lengths + [0] * (pages.sequences - users)))
        ids = torch.arange(pages.sequences, dtype=torch.int32, device=self.device)
        children = ids[users:users + total]
        pages.fork(ids[:total] // count, children)
        more = ((ids >= users) & (ids < users + total)).int()
        groups, shared = ids[:users + 1] * count, pages.lengths[:users]
        at = slice(users, users + total)
        u = uniforms.permute(2, 0, 1).contiguous()
        found = [sample(logits, u[0], return_logprobs=True, **settings)]
        settings = {name: x.repeat_interleave(count) if torch.is_tensor(x) else x
                    for name, x in settings.items()}

        def attend(cache, q):
            return cache.attend_shared(q, pages.table[at], pages.lengths[at], None, groups, shared,
                                       max_tokens=1)

        for step in range(1, steps):
            positions = pages.lengths[at].clone()
            pages.extend(more)
            logits = self._forward(found[-1][0].flatten(), positions,
                                   (pages.table[at], pages.lengths[at], None), 1, attend)
            drawn = sample(logits, u[step].view(total), return_logprobs=True, **settings)
            found.append([x.view(users, count) for x in drawn])
        pages.free(children)
        return tuple(torch.stack(x, -1) for x in zip(*found))

    def records(self, layer, user, start, count):
        """``count`` tokens of a user from ``start`` on as bf16 K || V records
        [count, kv_heads, 2 * head_dim]: what the window branch, the block
        summaries and the pool take."""
        if start < 0 or count < 0 or start + count > self.lengths[user]:
            raise ValueError("tokens past the user's history")
        table = self._tensor([self.pages[user] or [0]])
        k, v = self.caches[layer].read(table, self._tensor([start]), self._tensor([0, count]),
                                       total=count)
        return torch.cat((k, v), -1)

    def check(self):
        """Raise if a cache call met a page or length out of range."""
        for cache in self.caches:
            cache.check()
        if self.table:
            self.table.check()


def main():
    users, history, steps, candidates = 8, 4096, 16, 16
    model = DenseCacheModel(NSAConfig(layers=4), users=users, max_tokens=history + steps + 1,
                            candidates=candidates, candidate_tokens=steps)
    g = torch.Generator(device="cuda").manual_seed(0)
    prompt = torch.randint(0, model.cfg.vocab, (users * history,), generator=g, device="cuda")

    def timed(what, tokens, run):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        out = run()
        end.record()
        end.synchronize()
        ms = start.elapsed_time(end)
        print(f"{what}: {ms:.2f} ms, {tokens / ms * 1e3:.0f} tokens/s")
        return out

    last = torch.arange(1, users + 1, device="cuda") * history - 1
    logits = timed(f"prefill of {users} x {history}", users * history,
                   lambda: model.step(prompt, [history] * users)[last])

    def decode():
        nonlocal logits
        for _ in range(steps):
            logits = model.step(logits.argmax(-1), [1] * users)

    logits = model.step(logits.argmax(-1), [1] * users)
    timed(f"{steps} decode steps of {users} users", steps * users, decode)
    settings = dict(temperature=0.8, top_k=50, top_p=0.95)
    u = torch.rand(users, candidates, steps, generator=g, device="cuda")
    model.generate(logits, u, **settings)
    tokens, _ = timed(f"{steps} tokens of {candidates} candidates of {users} users",
                      steps * candidates * users, lambda: model.generate(logits, u, **settings))
    print(f"candidates: {tuple(tokens.shape)}")
    model.check()
    window = model.records(0, 0, history - 512, 512)
    print(f"window of user 0 read back: {tuple(window.shape)}")


if __name__ == "__main__":
    main()
