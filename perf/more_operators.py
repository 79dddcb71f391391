"""Measured cases of several continuations of one history over the dense 8-bit cache.

Four operators a program runs when candidates are generated from a user's long
history, which all of them share:

  fork     candidates of the last step dropped, new ones branched off their
           histories, a token's room taken for each
  compact  a pool with holes brought to the front, so that its rest can go
  shared   attention of the candidates' new tokens, the shared tokens read once
           for all candidates of a history
  sample   tokens drawn from the logits with temperature, top-k, top-p and min-p

The cache of one layer is ``codes [pages, kv heads, 2 (K, V), page, dim]`` in
8 bits and ``scales [pages, kv heads, 2]`` in fp32. A sequence's token t lies in
page ``table[b, t // page]`` at slot ``t % page``, in every layer; ``lengths[b]``
counts its tokens and ``references[p]`` the table entries that name page p.

``own`` chooses between the plain form (elementary torch operations) and the
framework's operators; ``exact`` gives the same results in fp64.
"""

import math

import numpy
import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
WIDTH = {"bf16": 2, "f16": 2, "f32": 4}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}   # largest code of a format

# ------------------------------------------------------------------ cases ---


def listed():
    return [
        # Four beams of one short history: the latency of a decode step.
        dict(name="shared beams", op="shared", groups=1, candidates=4, tokens=1, ragged=False,
             history=1000, own=5, heads=32, kv_heads=2, dim=64, page=64, format="e4m3",
             dtype="bf16", causal=True),
        # One new token of each of 64 candidates of one user's 16K history.
        dict(name="shared candidates", op="shared", groups=1, candidates=64, tokens=1,
             ragged=True, history=16384, own=8, heads=32, kv_heads=2, dim=64, page=64,
             format="e4m3", dtype="bf16", causal=True),
        # Eight users of unlike histories with up to 32 candidates each.
        dict(name="shared users", op="shared", groups=8, candidates=32, tokens=1, ragged=True,
             history=8191, own=40, heads=32, kv_heads=8, dim=128, page=32, format="int8",
             dtype="f16", causal=True),
        # Suffixes of 16 tokens of 16 candidates of two users: the extend step.
        dict(name="shared suffixes", op="shared", groups=2, candidates=16, tokens=16,
             ragged=False, history=16383, own=3, heads=32, kv_heads=2, dim=64, page=64,
             format="e4m3", dtype="bf16", causal=True),
        # One user's next token.
        dict(name="sample one", op="sample", rows=1, vocab=32000, dtype="bf16", draws=1,
             spread=2.5, temperature=0.8, top_k=50, top_p=0.95, min_p=0.0, mixed=False,
             masked=0.0),
        # A decode batch whose users each have their own settings.
        dict(name="sample batch", op="sample", rows=64, vocab=32000, dtype="bf16", draws=1,
             spread=2.5, temperature=0.9, top_k=200, top_p=0.9, min_p=0.02, mixed=True,
             masked=0.1),
        # The first tokens of 16 candidates from each of 8 users' logits, a large
        # vocabulary, nothing but top-p.
        dict(name="sample candidates", op="sample", rows=8, vocab=131071, dtype="f32", draws=16,
             spread=3.0, temperature=1.0, top_k=0, top_p=0.95, min_p=0.0, mixed=False,
             masked=0.0),
        # A large batch over the whole distribution.
        dict(name="sample large", op="sample", rows=256, vocab=128000, dtype="bf16", draws=1,
             spread=2.0, temperature=0.7, top_k=0, top_p=1.0, min_p=0.0, mixed=False,
             masked=0.0),
        # Beams of two users branched again.
        dict(name="fork beams", op="fork", groups=2, candidates=4, ragged=True, history=1000,
             layers=16, kv_heads=2, dim=64, page=64, format="e4m3", spare=100),
        # 256 candidates branched off four long histories.
        dict(name="fork candidates", op="fork", groups=4, candidates=64, ragged=True,
             history=16383, layers=4, kv_heads=8, dim=128, page=64, format="int8", spare=2000),
        # A small pool: most of what it held has gone.
        dict(name="compact small", op="compact", groups=5, candidates=2, history=700, layers=4,
             kv_heads=2, dim=64, page=16, format="int8", holes=0.7),
        # A pool of 64 users' histories, a third of the pages holes.
        dict(name="compact pool", op="compact", groups=64, candidates=1, history=4000, layers=2,
             kv_heads=8, dim=128, page=64, format="e4m3", holes=0.35),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("shared", "shared", "sample", "sample", "fork", "compact"))
    if op == "sample":
        rows = _spread(rng, 1, 256)
        return dict(op=op, rows=rows, vocab=_spread(rng, 500, min(131072, 32768000 // rows)),
                    dtype=rng.choice(("bf16", "f16", "f32")), draws=rng.choice((1, 1, 1, 2, 7, 16)),
                    spread=rng.uniform(1.0, 4.0), temperature=rng.choice((0.0, 0.5, 0.8, 1.0, 1.5)),
                    top_k=rng.choice((0, 0, 1, 20, 50, 1000)),
                    top_p=rng.choice((1.0, 1.0, 0.95, 0.9, 0.5)),
                    min_p=rng.choice((0.0, 0.0, 0.05, 0.1)), mixed=rng.random() < 0.5,
                    masked=rng.choice((0.0, 0.0, 0.1, 0.9)))
    kv_heads, dim = rng.choice(((2, 64), (2, 64), (8, 128), (4, 64), (1, 128)))
    case = dict(op=op, kv_heads=kv_heads, dim=dim, page=rng.choice((16, 32, 64)),
                format=rng.choice(("e4m3", "int8")))
    if op == "shared":
        groups = _spread(rng, 1, 8)
        tokens = rng.choice((1, 1, 1, 2, 5, 16))
        return dict(case, groups=groups, tokens=tokens,
                    candidates=_spread(rng, 1, max(1, 256 // (groups * tokens))),
                    ragged=rng.random() < 0.7, history=_spread(rng, 64, 16384 // groups),
                    own=_spread(rng, 1, 200) - 1, heads=kv_heads * rng.choice((1, 4, 32 // kv_heads)),
                    dtype=rng.choice(("bf16", "f16")), causal=rng.random() < 0.8)
    if op == "fork":
        groups = _spread(rng, 1, 8)
        return dict(case, groups=groups, candidates=_spread(rng, 1, 256 // groups),
                    ragged=rng.random() < 0.7, history=_spread(rng, 10, 32768 // groups),
                    layers=rng.choice((1, 3, 4, 16)) if kv_heads < 8 else rng.choice((1, 3, 4)),
                    spare=_spread(rng, 1, 2000))
    groups = _spread(rng, 1, 64)
    return dict(case, groups=groups, candidates=_spread(rng, 1, max(1, 64 // groups)),
                history=_spread(rng, 10, 4000), layers=rng.choice((1, 2)),
                holes=rng.uniform(0.05, 0.9))


def _counts(case):
    """Candidates of each history."""
    n, top = case["groups"], case["candidates"]
    if not case.get("ragged"):
        return [top] * n
    return [max(1, top - (g * 2654435761 >> 7) % top) if g else top for g in range(n)]


def _histories(case):
    """Tokens of each history; unlike ones unless there is but one."""
    n, top = case["groups"], case["history"]
    if not case.get("ragged", True):
        return [top] * n
    return [top - (g * 2246822519 >> 5) % (top // 2 + 1) if g else top for g in range(n)]


def _candidates(case):
    """(history, own tokens before the new ones, new tokens) of each candidate."""
    found = []
    for g, n in enumerate(_counts(case)):
        for i in range(n):
            own_, new = case["own"], case["tokens"]
            if case["ragged"]:
                own_ -= (i * 2654435761 >> 9) % (own_ + 1)
                new -= (i * 2246822519 >> 11) % new if i else 0
            found.append((g, own_, new))
    return found


def _page_bytes(case):
    return 2 * case["kv_heads"] * (case["page"] * case["dim"] + 4)


def work(case):
    if case["op"] == "sample":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * WIDTH[case["dtype"]] + 20 * case["rows"] * case["draws"],
                "flops": 2 * values}
    page = case["page"]
    if case["op"] == "shared":
        dim, kv, heads = case["dim"], case["kv_heads"], case["heads"]
        histories = _histories(case)
        cached, rows, pairs = sum(histories), 0, 0
        for g, own_, new in _candidates(case):
            cached += own_ + new
            rows += new
            pairs += new * (histories[g] + own_ + new)
            if case["causal"]:
                pairs -= new * (new - 1) // 2
        return {"bytes": 2 * dim * kv * cached + -(-cached // page) * (8 * kv + 4)
                + rows * heads * (2 * dim * WIDTH[case["dtype"]] + 4),
                "flops": 4 * dim * heads * pairs}
    if case["op"] == "fork":
        copied = sum(n * (h % page) * 2 * case["kv_heads"] * case["dim"]
                     for n, h in zip(_counts(case), _histories(case)))
        shared = sum(n * (-(-h // page)) for n, h in zip(_counts(case), _histories(case)))
        return {"bytes": 2 * case["layers"] * copied + 12 * shared, "flops": 0}
    pages, live = _sizes(case)
    # About as many pages move as there are live ones past the first `live` ids.
    moved = live * (pages - live) // pages
    return {"bytes": 2 * case["layers"] * moved * _page_bytes(case) + 8 * pages, "flops": 0}


# ----------------------------------------------------------------- inputs ---


def _sizes(case):
    """(pages of the pool, pages in use) of a pool to compact."""
    page, live = case["page"], 0
    for h in _histories(case):
        live += h // page + (case["candidates"] if h % page else 0)
    return max(live + 1, round(live / (1 - case["holes"]))), live


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _pool(case, g, pages, layers):
    """Pages of every layer, all of them with some tokens' codes."""
    kv, page, dim = case["kv_heads"], case["page"], case["dim"]
    codes, scales = [], []
    for _ in range(layers):
        if case["format"] == "e4m3":  # normal values; the page's largest is the largest code
            c = torch.empty(pages, kv, 2, page, dim, dtype=torch.uint8, device=DEVICE)
            for low in range(0, pages, 512):
                part = c[low:low + 512]
                x = torch.randn(part.shape, generator=g, device=DEVICE)
                x *= TOP["e4m3"] / x.abs().amax((-2, -1), keepdim=True)
                part.copy_(x.to(torch.float8_e4m3fn).view(torch.uint8))
        else:
            c = torch.randint(-127, 128, (pages, kv, 2, page, dim), generator=g, device=DEVICE,
                              dtype=torch.int8)
        codes.append(c.view(CODES[case["format"]]))
        scales.append(torch.exp(0.5 * torch.randn(pages, kv, 2, generator=g, device=DEVICE))
                      * (3.0 / TOP[case["format"]]))
    return codes, scales


def _order(seed, pages):
    return torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()


def _padded(rows, width):
    return _ints([r + [-1] * (width - len(r)) for r in rows])


def _shared(case, g, seed, state):
    """Candidates over histories: the full pages of a history are in every
    candidate's row, its partly filled one is each candidate's own copy."""
    page, histories, found = case["page"], _histories(case), _candidates(case)
    full = [h // page for h in histories]
    tail = [-(-(histories[c] + o + n) // page) - full[c] for c, o, n in found]
    order = _order(seed, sum(full) + sum(tail) + 2)
    (codes,), (scales,) = _pool(case, g, len(order), 1)
    history = [[order.pop() for _ in range(n)] for n in full]
    rows, first, copies = [], {}, []
    for (c, _, _), n in zip(found, tail):
        mine = [order.pop() for _ in range(n)]
        if histories[c] % page and first.setdefault(c, mine[0]) != mine[0]:
            copies.append((first[c], mine[0], histories[c] % page))
        rows.append(history[c] + mine)
    for source, target, fill in copies:
        codes.view(torch.uint8)[target, :, :, :fill] = codes.view(torch.uint8)[source, :, :, :fill]
        scales[target] = scales[source]
    counts, offsets, groups = _counts(case), [0], [0]
    for _, _, n in found:
        offsets.append(offsets[-1] + n)
    for n in counts:
        groups.append(groups[-1] + n)
    state.update(codes=codes, scales=scales, table=_padded(rows, max(map(len, rows))),
                 lengths=_ints([histories[c] + o + n for c, o, n in found]),
                 offsets=_ints(offsets), groups=_ints(groups), shared=_ints(histories),
                 max_tokens=max(n for _, _, n in found), scale=case["dim"] ** -0.5)
    q = torch.randn(offsets[-1], case["heads"], case["dim"], generator=g, device=DEVICE)
    state["q"] = q.to(TYPES[case["dtype"]])
    if own:
        from cxlsparse_b200.quantized import QuantizedCache

        state["cache"] = QuantizedCache(codes=codes, scales=scales)


def _sample(case, g, state):
    rows, vocab = case["rows"], case["vocab"]
    logits = case["spread"] * torch.randn(rows, vocab, generator=g, device=DEVICE)
    # A few likely tokens, as a trained model has.
    likely = torch.randint(0, vocab, (rows, 20), generator=g, device=DEVICE)
    logits.scatter_add_(1, likely, 3 * case["spread"] * torch.rand(rows, 20, generator=g,
                                                                   device=DEVICE))
    if case["masked"]:
        hidden = torch.rand(rows, vocab, generator=g, device=DEVICE) < case["masked"]
        logits.masked_fill_(hidden, -math.inf)
    state["logits"] = logits.to(TYPES[case["dtype"]])
    shape = (rows, case["draws"]) if case["draws"] > 1 else (rows,)
    state["uniforms"] = torch.rand(shape, generator=g, device=DEVICE)
    row = torch.arange(rows, device=DEVICE)

    def each(value, other):
        """One value for all, or some rows' own."""
        if not case["mixed"]:
            return value
        kind = torch.int32 if isinstance(value, int) else torch.float32
        return torch.where(row % 4 == 1, other, value).to(kind)

    state.update(temperature=each(case["temperature"], 0.6), top_k=each(case["top_k"], 0),
                 top_p=each(case["top_p"], 1.0), min_p=each(case["min_p"], 0.1))


def _fork(case, g, seed, state):
    """Histories in sequences 0 .., their candidates behind them, forked once."""
    page, histories, counts = case["page"], _histories(case), _counts(case)
    children = sum(counts)
    held = sum(-(-h // page) for h in histories)
    order = _order(seed, held + 2 * children + case["spare"])
    codes, scales = _pool(case, g, len(order), case["layers"])
    rows = [[order.pop() for _ in range(-(-h // page))] for h in histories]
    parents = [c for c, n in enumerate(counts) for _ in range(n)]
    references = [0] * (len(order) + held)
    for r in rows:
        for p in r:
            references[p] += 1
    n = len(rows) + children
    width = max(map(len, rows)) + 2
    state.update(codes=codes, scales=scales,
                 table=_padded(rows + [[]] * children, width),
                 lengths=_ints(histories + [0] * children), references=_ints(references),
                 parents=_ints(parents), children=_ints(range(len(rows), n)),
                 more=_ints([0] * len(rows) + [1] * children))


def _compact(case, g, seed, state):
    page, (pages, live) = case["page"], _sizes(case)
    order = _order(seed, pages)
    codes, scales = _pool(case, g, pages, case["layers"])
    rows, lengths = [], []
    for h in _histories(case):
        full = [order.pop() for _ in range(h // page)]
        for _ in range(case["candidates"]):
            rows.append(full + ([order.pop()] if h % page else []))
            lengths.append(h)
    width = max(1, max(map(len, rows)))
    state.update(codes=codes, scales=scales, given=_padded(rows, width),
                 given_lengths=_ints(lengths),
                 table=torch.full((len(rows), width), -1, dtype=torch.int32, device=DEVICE),
                 lengths=torch.zeros(len(rows), dtype=torch.int32, device=DEVICE),
                 references=torch.zeros(pages, dtype=torch.int32, device=DEVICE))


def prepare(case, seed):
    g, state = _generator(seed), dict(case=case)
    if case["op"] == "sample":
        _sample(case, g, state)
        return state
    if case["op"] == "shared":
        _shared(case, g, seed, state)
        return state
    (_fork if case["op"] == "fork" else _compact)(case, g, seed, state)
    if own:
        from cxlsparse_b200.pages import PageTable
        from cxlsparse_b200.quantized import QuantizedCache

        caches = [QuantizedCache(codes=c, scales=s)
                  for c, s in zip(state["codes"], state["scales"])]
        sequences, width = state["table"].shape
        state["pages"] = PageTable(caches, sequences, width)
        if case["op"] == "fork":
            state["pages"].adopt(state["table"], state["lengths"])
    return state


# -------------------------------------------------------------- one pass ---


def run(state):
    case = state["case"]
    if not own:
        return {"shared": _plain_shared, "sample": _plain_sample, "fork": _plain_fork,
                "compact": _plain_compact}[case["op"]](state, case)
    if case["op"] == "shared":
        out, lse = state["cache"].attend_shared(
            state["q"], state["table"], state["lengths"], state["offsets"], state["groups"],
            state["shared"], max_tokens=state["max_tokens"], causal=case["causal"],
            scale=state["scale"], return_lse=True)
        return {"out": out, "lse": lse}
    if case["op"] == "sample":
        from cxlsparse_b200.sampling import sample

        tokens, logprobs = sample(
            state["logits"], state["uniforms"], temperature=state["temperature"],
            top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"],
            return_logprobs=True)
        return {"tokens": tokens, "logprobs": logprobs}
    pages = state["pages"]
    if case["op"] == "fork":
        pages.free(state["children"])
        pages.fork(state["parents"], state["children"])
        pages.extend(state["more"])
    else:
        pages.adopt(state["given"], state["given_lengths"])
        pages.compact()
    return {"table": pages.table, "lengths": pages.lengths, "references": pages.references,
            "codes": state["codes"], "scales": state["scales"]}


# The plain forms: fp32, and fp64 for what lies next to a border.


def _rows(state, case, users, position):
    """K and V [users, n, kv heads, dim] at `position` [n] or [users, n]."""
    page, table = case["page"], state["table"][users]
    position = position.expand(len(table), -1)
    block = (position // page).clamp(0, table.shape[1] - 1)
    pages = table.gather(1, block).long().clamp(min=0)
    codes = state["codes"].view(torch.uint8)[pages, :, :, position % page]
    values = codes.view(state["codes"].dtype).float() * state["scales"][pages][..., None]
    return values[:, :, :, 0], values[:, :, :, 1]


def _plain_shared(state, case):
    q, most = state["q"], state["max_tokens"]
    kv, dim, group = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    groups, shared = state["groups"].tolist(), state["shared"].tolist()
    offsets, lengths = state["offsets"], state["lengths"]
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=q.device)
    for c, size in enumerate(shared):
        users = torch.arange(groups[c], groups[c + 1], device=q.device)
        first, count = offsets[users].long(), (offsets[users + 1] - offsets[users]).long()
        step = torch.arange(most, device=q.device)
        real = step < count[:, None]                                  # [users, most]
        at = (first[:, None] + step).clamp(max=len(q) - 1)
        x = q[at].float().view(len(users), most, kv, group, dim)
        # The shared keys, once for all rows.
        k, v = _rows(state, case, users[:1], torch.arange(size, device=q.device)[None])
        s = torch.einsum("umhgd,khd->humgk", x, k[0]) * state["scale"]
        m1 = s.amax(-1)
        p = (s - m1[..., None]).exp_()
        l1, o1 = p.sum(-1), torch.einsum("humgk,khd->humgd", p, v[0])
        # Each candidate's own.
        width = state["table"].shape[1] * case["page"] - size
        key = size + torch.arange(width, device=q.device)[None]
        k, v = _rows(state, case, users, key)
        s = torch.einsum("umhgd,ukhd->humgk", x, k) * state["scale"]
        position = (lengths[users] - count)[:, None] + step
        seen = (key < lengths[users, None])[:, None]                  # [users, 1, keys]
        if case["causal"]:
            seen = seen & (key[:, None] <= position[..., None])
        s = s.masked_fill(~seen[None, :, :, None], -math.inf)
        m = torch.maximum(m1, s.amax(-1))
        p = (s - m[..., None]).exp_()
        v = torch.where((key < lengths[users, None])[..., None, None], v, 0.0)
        f = (m1 - m).exp()
        total = l1 * f + p.sum(-1)
        o = o1 * f[..., None] + torch.einsum("humgk,ukhd->humgd", p, v)
        o = (o / total[..., None]).permute(1, 2, 0, 3, 4).flatten(2, 3)
        out[at[real]] = o[real].to(q.dtype)
        lse[at[real]] = (m + total.log()).permute(1, 2, 0, 3).flatten(2, 3)[real]
    return {"out": out, "lse": lse}


def _plain_sample(state, case):
    x = state["logits"].double()
    rows, vocab = x.shape

    def column(value):
        return torch.as_tensor(value, device=x.device).expand(rows)[:, None]

    temperature = column(state["temperature"]).float().double()
    top_k, greedy = column(state["top_k"]), temperature == 0
    top_p = column(state["top_p"]).float().double()
    min_p = column(state["min_p"]).float().double()
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    s = x.gather(1, order)
    top = s[:, :1]
    w = ((s - top) / torch.where(greedy, 1.0, temperature)).exp()
    rank = torch.arange(vocab, device=x.device)
    keep = (top_k <= 0) | (rank < top_k)
    keep &= (min_p <= 0) | greedy | (s - top >= temperature * min_p.log())
    keep &= ~greedy | (rank < 1)
    w = torch.where(keep, w, 0.0)
    before = w.cumsum(-1) - w
    keep &= (top_p >= 1) | (before < top_p * w.sum(-1, keepdim=True)) | (rank < 1)
    mass = torch.zeros_like(x).scatter_(1, order, torch.where(keep, w, 0.0)).cumsum(-1)
    u = state["uniforms"].double().view(rows, -1)
    tokens = torch.searchsorted(mass, u * mass[:, -1:], right=True)
    weight = (x - top).exp().sum(-1, keepdim=True).log()
    logprobs = (x.gather(1, tokens) - top - weight).float()
    shape = state["uniforms"].shape
    return {"tokens": tokens.view(shape), "logprobs": logprobs.view(shape)}


def _lowest_free(references, n):
    return torch.nonzero(references == 0)[:n, 0].to(torch.int32)


def _count(table, pages):
    flat = table.flatten().long()
    return torch.bincount(flat[flat >= 0], minlength=pages).to(torch.int32)


def _copy(state, source, target, fill):
    """Slots below fill[i] of page source[i] into page target[i], in every layer."""
    page = state["case"]["page"]
    slot = (torch.arange(page, device=fill.device) < fill[:, None])[:, None, None, :, None]
    source, target = source.long(), target.long()
    for codes, scales in zip(state["codes"], state["scales"]):
        c = codes.view(torch.uint8)
        c[target] = torch.where(slot, c[source], c[target])
        scales[target] = scales[source]


def _plain_fork(state, case):
    page, table, lengths = case["page"], state["table"], state["lengths"]
    children, parents = state["children"].long(), state["parents"].long()
    references = state["references"]
    # The last step's candidates go,
    table[children] = -1
    lengths[children] = 0
    references.copy_(_count(table, len(references)))
    # new ones take their histories' full pages and a copy of the last one,
    size = lengths[parents]
    block = torch.arange(table.shape[1], device=table.device)
    rows = torch.where(block < (size // page)[:, None], table[parents], -1)
    part = torch.nonzero(size % page)[:, 0]
    fresh = _lowest_free(references, len(part))
    at = (size // page)[part].long()
    _copy(state, table[parents[part], at], fresh, (size % page)[part])
    rows[part, at] = fresh
    table[children] = rows
    lengths[children] = size
    references.copy_(_count(table, len(references)))
    # and a page for the next token where the last one is full.
    after = lengths + state["more"]
    need = torch.nonzero((after + page - 1) // page > (lengths + page - 1) // page)[:, 0]
    fresh = _lowest_free(references, len(need))
    table[need, ((lengths + page - 1) // page)[need].long()] = fresh
    lengths.copy_(after)
    references.copy_(_count(table, len(references)))
    return {k: state[k] for k in ("table", "lengths", "references", "codes", "scales")}


def _plain_compact(state, case):
    table, lengths, references = state["table"], state["lengths"], state["references"]
    table.copy_(state["given"])
    lengths.copy_(state["given_lengths"])
    references.copy_(_count(table, len(references)))
    used = references > 0
    live = int(used.sum())
    source = live + torch.nonzero(used[live:])[:, 0]
    target = torch.nonzero(~used[:live])[:, 0]
    moved = torch.arange(len(references), device=table.device, dtype=torch.int32)
    moved[source] = target.to(torch.int32)
    for codes, scales in zip(state["codes"], state["scales"]):
        c = codes.view(torch.uint8)
        c[target] = c[source]
        scales[target] = scales[source]
    table.copy_(torch.where(table >= 0, moved[table.clamp(min=0).long()], -1))
    references[target] = references[source]
    references[source] = 0
    return {k: state[k] for k in ("table", "lengths", "references", "codes", "scales")}


# ------------------------------------------------------------- in 64 bits ---


def exact(case, seed):
    if case["op"] == "shared":
        pairs = work(case)["flops"]
        if pairs > 2e12:
            return None
    elif case["op"] == "sample" and case["rows"] * case["vocab"] > 2 ** 25:
        return None
    state = prepare(case, seed)
    return {"shared": _exact_shared, "sample": _exact_sample, "fork": _exact_pages,
            "compact": _exact_pages}[case["op"]](state, case)


def _exact_shared(state, case):
    """Every candidate on its own, over its own row of pages."""
    table, lengths = state["table"].tolist(), state["lengths"].tolist()
    offsets, page = state["offsets"].tolist(), case["page"]
    outs, lses = [], []
    for b, length in enumerate(lengths):
        ids = table[b][:-(-length // page)]
        held = state["codes"].view(torch.uint8)[ids].view(state["codes"].dtype).double()
        held = held * state["scales"][ids].double()[..., None, None]
        k, v = held.permute(2, 1, 0, 3, 4).flatten(2, 3)[:, :, :length]
        n = offsets[b + 1] - offsets[b]
        q = state["q"][offsets[b]:offsets[b + 1]].double()
        q = q.view(n, case["kv_heads"], -1, case["dim"])
        s = torch.einsum("nhgd,hkd->nhgk", q, k) * state["scale"]
        if case["causal"]:
            late = torch.arange(length, device=DEVICE) > torch.arange(length - n, length,
                                                                      device=DEVICE)[:, None]
            s = s.masked_fill(late[:, None, None], -math.inf)
        m = torch.logsumexp(s, -1)
        outs.append(torch.einsum("nhgk,hkd->nhgd", torch.exp(s - m[..., None]), v).flatten(1, 2))
        lses.append(m.flatten(1, 2))
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def _exact_sample(state, case):
    rows = case["rows"]

    def each(value):
        if torch.is_tensor(value):
            return value.double().tolist()
        return [float(numpy.float32(value))] * rows

    settings = list(zip(*(each(state[k]) for k in ("temperature", "top_k", "top_p", "min_p"))))
    logits = state["logits"].double().cpu().numpy()
    u = state["uniforms"].double().view(rows, -1).cpu().numpy()
    tokens = numpy.zeros(u.shape)
    logprobs = numpy.zeros(u.shape)
    for r, (temperature, top_k, top_p, min_p) in enumerate(settings):
        x = logits[r]
        top = x.max()
        total = numpy.exp(x - top).sum()
        if temperature == 0:
            tokens[r] = x.argmax()
        else:
            order = numpy.lexsort((numpy.arange(len(x)), -x))
            if top_k:
                order = order[:int(top_k)]
            p = numpy.exp((x[order] - top) / temperature)
            kept = p >= min_p * (1 - 1e-15)
            order, p = order[kept], p[kept]
            if top_p < 1:
                sums = numpy.cumsum(p)
                n = max(1, int(((sums - p) < top_p * sums[-1]).sum()))
                order, p = order[:n], p[:n]
            back = numpy.argsort(order)
            order, p = order[back], p[back]
            sums = numpy.cumsum(p)
            at = numpy.searchsorted(sums, u[r] * sums[-1], side="right")
            tokens[r] = order[numpy.minimum(at, len(order) - 1)]
        logprobs[r] = x[tokens[r].astype(int)] - top - math.log(total)
    shape = tuple(state["uniforms"].shape)
    return {"tokens": torch.from_numpy(tokens).view(shape),
            "logprobs": torch.from_numpy(logprobs).view(shape)}


def _exact_pages(state, case):
    """Page by page on the host; the codes follow the list of copies."""
    page = case["page"]
    compact = case["op"] == "compact"
    table = (state["given"] if compact else state["table"]).tolist()
    lengths = (state["given_lengths"] if compact else state["lengths"]).tolist()
    uses = {}
    for row in table:
        for p in row:
            if p >= 0:
                uses[p] = uses.get(p, 0) + 1
    copies = []                                  # (source, target, slots)
    if compact:
        live = len(uses)
        holes = [p for p in range(live) if p not in uses]
        names = dict(zip(sorted(p for p in uses if p >= live), holes))
        copies = [(s, t, page) for s, t in names.items()]
        table = [[names.get(p, p) for p in row] for row in table]
    else:
        taken, lowest = set(uses), 0
        grown = state["more"].tolist()

        def take():
            nonlocal lowest
            while lowest in taken:
                lowest += 1
            taken.add(lowest)
            return lowest

        for parent, child in zip(state["parents"].tolist(), state["children"].tolist()):
            length = lengths[parent]
            row = [p if j < length // page else -1 for j, p in enumerate(table[parent])]
            if length % page:
                row[length // page] = take()
                copies.append((table[parent][length // page], row[length // page], length % page))
            table[child], lengths[child] = row, length
        for b, n in enumerate(grown):
            for t in range(lengths[b], lengths[b] + n):
                if t % page == 0:
                    table[b][t // page] = take()
            lengths[b] += n
    references = [0] * len(state["references"])
    for row in table:
        for p in row:
            if p >= 0:
                references[p] += 1
    found = {"table": table, "lengths": lengths, "references": references}
    found = {k: torch.tensor(v, dtype=torch.float64) for k, v in found.items()}
    codes, scales = [], []
    for c, s in zip(state["codes"], state["scales"]):
        c, s = c.view(torch.uint8).clone(), s.clone()
        for source, target, slots in copies:
            c[target, :, :, :slots] = c[source, :, :, :slots]
            s[target] = s[source]
        codes.append(None)                       # bytes of a format: no value in 64 bits
        scales.append(s.double())
    found.update(codes=codes, scales=scales)
    return found
