"""Measured cases of the dense 8-bit key/value cache and its rotary positions.

Four operators a program runs per layer when a user's whole history is kept in
HBM at 8 bits a channel:

  rotary  rotary positions of queries and keys (or, transposed, their gradient)
  append  new tokens' keys and values quantised into the pages of the cache
  read    tokens of the cache brought back to 16 or 32 bits
  attend  attention of new queries over the cached tokens

The cache of one layer is ``codes [pages, kv heads, 2 (K, V), page, dim]`` in
8 bits and ``scales [pages, kv heads, 2]`` in fp32, a scale for each page of
tokens, head and part. A sequence's token t lies in page ``table[b, t // page]``
at slot ``t % page``. ``lengths[b]`` counts its tokens, the new ones included;
the new tokens of sequence b are rows ``offsets[b] .. offsets[b + 1]`` of the
packed inputs.

``own`` chooses between the plain form (elementary torch operations in fp32)
and the framework's operators; ``exact`` gives the same results in fp64.
"""

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
WIDTH = {"bf16": 2, "f16": 2, "f32": 4}
TOP = {"e4m3": 448.0, "int8": 127.0}   # largest code of a format
LEAST = 2.0 ** -64                     # smallest scale of a page

# ------------------------------------------------------------------ cases ---


def listed():
    return [
        # One new token of each of eight users: the latency of a decode step.
        dict(name="rotary decode", op="rotary", users=8, tokens=1, ragged=False, heads=32,
             kv_heads=2, dim=64, rotary=64, layout="half", scaling="none", dtype="bf16",
             transpose=False, fused=True, last=16384),
        # A prefill of four long documents, interleaved pairs over half of the
        # head, frequencies stretched for a longer context.
        dict(name="rotary prefill", op="rotary", users=4, tokens=8191, ragged=True, heads=32,
             kv_heads=8, dim=128, rotary=64, layout="interleaved", scaling="yarn", dtype="f16",
             transpose=False, fused=False, last=131072),
        # The gradient of the rotary step of a training batch, in fp32.
        dict(name="rotary gradient", op="rotary", users=2, tokens=2048, ragged=False, heads=32,
             kv_heads=2, dim=64, rotary=64, layout="half", scaling="linear", dtype="f32",
             transpose=True, fused=False, last=2048),
        # One new token of each of eight users into partly filled pages.
        dict(name="append decode", op="append", users=8, tokens=1, ragged=True, history=4096,
             kv_heads=2, dim=64, page=64, format="e4m3", dtype="bf16", fused=True),
        # Suffixes of odd lengths, starting and ending inside pages.
        dict(name="append suffixes", op="append", users=5, tokens=301, ragged=True, history=1000,
             kv_heads=8, dim=128, page=32, format="int8", dtype="f16", fused=False),
        # A prefill of four histories into empty pages.
        dict(name="append prefill", op="append", users=4, tokens=8192, ragged=False, history=0,
             kv_heads=8, dim=128, page=64, format="e4m3", dtype="bf16", fused=False),
        # The sliding window of one user, out of the middle of a page.
        dict(name="read window", op="read", users=1, tokens=511, ragged=False, history=4001,
             kv_heads=2, dim=64, page=64, format="e4m3", dtype="bf16"),
        # Whole histories, for a kernel that takes 16 bits.
        dict(name="read histories", op="read", users=4, tokens=16384, ragged=True, history=0,
             kv_heads=8, dim=128, page=64, format="int8", dtype="f16"),
        # One user's next token over a 4K history.
        dict(name="attend one token", op="attend", users=1, tokens=1, ragged=False, history=4096,
             heads=32, kv_heads=2, dim=64, page=64, format="e4m3", dtype="bf16", causal=True,
             window=0),
        # A decode batch of 64 users, histories from none to 16K.
        dict(name="attend decode batch", op="attend", users=64, tokens=1, ragged=True,
             history=16384, heads=32, kv_heads=2, dim=64, page=64, format="e4m3", dtype="bf16",
             causal=True, window=0),
        # A 256-token suffix over a 16K history: the extend step.
        dict(name="attend extend", op="attend", users=1, tokens=256, ragged=False, history=16384,
             heads=32, kv_heads=2, dim=64, page=64, format="e4m3", dtype="bf16", causal=True,
             window=0),
        # A prefill chunk of three users, wider heads, 8-bit integers.
        dict(name="attend prefill chunk", op="attend", users=3, tokens=1999, ragged=True,
             history=6001, heads=32, kv_heads=8, dim=128, page=64, format="int8", dtype="f16",
             causal=True, window=0),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("rotary", "append", "read", "attend", "attend"))
    heads, kv_heads = rng.choice(((32, 2), (32, 8), (32, 8), (8, 8), (12, 4), (16, 1)))
    case = dict(op=op, ragged=rng.random() < 0.7, kv_heads=kv_heads,
                dim=rng.choice((64, 128)))
    if op == "rotary":
        users = _spread(rng, 1, 16)
        dim = case["dim"]
        return dict(case, users=users, tokens=_spread(rng, 1, 8191 // users), heads=heads,
                    rotary=rng.choice((dim, dim, dim // 2, dim - 16)),
                    layout=rng.choice(("half", "interleaved")),
                    scaling=rng.choice(("none", "linear", "ntk", "yarn")),
                    dtype=rng.choice(("bf16", "f16", "f32")), transpose=rng.random() < 0.5,
                    fused=rng.random() < 0.5, last=_spread(rng, 8192, 131072))
    case.update(page=rng.choice((16, 32, 64)), format=rng.choice(("e4m3", "int8")))
    if op == "append":
        users = _spread(rng, 1, 16)
        return dict(case, users=users, tokens=_spread(rng, 1, 16384 // users),
                    history=_spread(rng, 1, 8192) - 1, dtype=rng.choice(("bf16", "f16", "f32")),
                    fused=rng.random() < 0.5)
    if op == "read":
        users = _spread(rng, 1, 16)
        return dict(case, users=users, tokens=_spread(rng, 1, 32768 // users),
                    history=_spread(rng, 1, 8192) - 1, dtype=rng.choice(("bf16", "f16", "f32")))
    case.update(heads=heads, dtype=rng.choice(("bf16", "f16")), causal=rng.random() < 0.8,
                window=rng.choice((0, 0, 0, 512, 4095)))
    if rng.random() < 0.6:                       # decode: one to eight tokens
        users = _spread(rng, 1, 64)
        return dict(case, users=users, tokens=rng.choice((1, 1, 1, 2, 5, 8)),
                    history=_spread(rng, 64, 524288 // max(users, 32)))
    users = _spread(rng, 1, 4)                   # a suffix or a prefill chunk
    return dict(case, users=users, tokens=_spread(rng, 9, 1024 // users),
                history=_spread(rng, 64, 16384 // users) - 1)


def _tokens(case):
    """New tokens of each sequence (at least one)."""
    n, top = case["users"], case["tokens"]
    if not case["ragged"]:
        return [top] * n
    return [max(1, top - (i * 2654435761 >> 7) % max(1, top)) if i else top for i in range(n)]


def _history(case):
    """Tokens of each sequence before the new ones (one sequence of a large
    ragged batch has none)."""
    n, top = case["users"], case["history"]
    if not case["ragged"]:
        return [top] * n
    return [0 if i == 3 else top - (i * 2246822519 >> 5) % (top + 1) if i else top
            for i in range(n)]


def _pairs(case):
    """(query, key) pairs of one head that attention looks at."""
    total, window = 0, case["window"]
    for new, old in zip(_tokens(case), _history(case)):
        length = old + new
        for position in range(old, length):
            high = position + 1 if case["causal"] else length
            low = max(0, position - window + 1) if window else 0
            total += high - low
    return total


def work(case):
    new, dim, kv = sum(_tokens(case)), case["dim"], case["kv_heads"]
    width = WIDTH[case["dtype"]]
    if case["op"] == "rotary":
        rows = new * (case["heads"] + kv)
        return {"bytes": 2 * rows * dim * width + 4 * new, "flops": 3 * rows * case["rotary"]}
    pages = sum(-(-(o + n) // case["page"]) - o // case["page"]
                for n, o in zip(_tokens(case), _history(case)))
    if case["op"] == "append":
        values = 2 * new * kv * dim
        return {"bytes": values * (width + 1) + pages * (8 * kv + 4), "flops": 2 * values}
    if case["op"] == "read":
        values = 2 * new * kv * dim
        return {"bytes": values * (width + 1) + pages * (8 * kv + 4), "flops": values}
    rows = new * case["heads"]
    cached = 0
    for n, o in zip(_tokens(case), _history(case)):
        low = max(0, o - case["window"] + 1) if case["window"] else 0
        cached += o + n - low
    pages = -(-cached // case["page"])
    return {"bytes": rows * (2 * dim * width + 4) + cached * kv * 2 * dim + pages * (8 * kv + 4),
            "flops": 4 * dim * case["heads"] * _pairs(case)}


# ----------------------------------------------------------------- inputs ---


def _frequencies(case):
    """Radians per position of every pair, fp64, and the magnitude of the
    rotation: theta 10000; linear: positions divided by 4; ntk: theta raised so
    that the slowest pair is stretched 4 times; yarn (Peng et al. 2023): pairs
    below one turn per 4096 positions stretched 4 times, pairs above 32 turns
    kept, a ramp between them, magnitude 0.1 ln 4 + 1."""
    d, theta, factor, original = case["rotary"], 10000.0, 4.0, 4096
    if case["scaling"] == "ntk":
        theta *= factor ** (d / (d - 2))
    index = torch.arange(0, d, 2, dtype=torch.float64)
    f = theta ** (-index / d)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "yarn":
        def pair(turns):
            return d * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(0, math.floor(pair(32))), min(d - 1, math.ceil(pair(1)))
        ramp = ((index / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1
    return f, 1.0


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEVICE).to(dtype)


def _offsets(counts):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32,
                        device=DEVICE)


def _to_codes(case, x):
    """Values in units of the scale -> codes (round to nearest even, saturated)."""
    x = x.clamp(-TOP[case["format"]], TOP[case["format"]])
    if case["format"] == "e4m3":
        return x.to(torch.float8_e4m3fn)
    return torch.nan_to_num(x, nan=0.0).round().to(torch.int8)


def _cache(case, g, lengths, new, written):
    """A cache that holds the first `written` tokens of each sequence; what no
    token was written to holds whatever the pool's memory held."""
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    need = [-(-n // page) for n in lengths]
    pages, width = sum(need) + 3, max(max(need), 1)
    order = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    # Channels of different size, as keys have; values of a few pages far larger.
    channel = torch.exp(0.5 * _normal(g, kv, 2, 1, dim))
    values = _normal(g, pages, kv, 2, page, dim) * channel
    values *= torch.exp(0.7 * _normal(g, pages, kv, 2, 1, 1))
    scales = (values.abs().amax((-2, -1)) * (1 / TOP[case["format"]])).clamp(min=LEAST)
    codes = _to_codes(case, values / scales[..., None, None]).view(torch.uint8)
    count = torch.tensor(written, device=DEVICE)
    slots = torch.arange(width * page, device=DEVICE).view(1, width, page)
    empty = slots >= count.view(-1, 1, 1)                       # [users, width, page]
    hole = torch.ones(pages, page, dtype=torch.bool, device=DEVICE)
    known = table >= 0
    hole[table[known].long()] = empty[known]
    codes.masked_fill_(hole[:, None, None, :, None], 0x7F)
    scales.masked_fill_(hole.all(1)[:, None, None], math.nan)
    return dict(codes=codes.view(torch.float8_e4m3fn if case["format"] == "e4m3"
                                 else torch.int8), scales=scales, table=table)


def prepare(case, seed):
    g = _generator(seed)
    dtype, dim, kv = TYPES[case["dtype"]], case["dim"], case["kv_heads"]
    new = _tokens(case)
    total = sum(new)
    state = dict(case=case, max_tokens=max(new))
    if case["op"] == "rotary":
        heads = case["heads"]
        if case["fused"]:  # slices of one projection's output
            proj = _normal(g, total, (heads + 2 * kv) * dim, dtype=dtype)
            state["q"] = proj[:, :heads * dim].view(total, heads, dim)
            state["k"] = proj[:, heads * dim:(heads + kv) * dim].view(total, kv, dim)
        else:
            state["q"] = _normal(g, total, heads, dim, dtype=dtype)
            state["k"] = _normal(g, total, kv, dim, dtype=dtype)
        first = torch.randint(0, max(1, case["last"] - max(new) + 1), (case["users"],),
                              generator=g, device=DEVICE)
        first = torch.repeat_interleave(first, torch.tensor(new, device=DEVICE))
        within = torch.cat([torch.arange(n) for n in new]).to(DEVICE)
        state["positions"] = (first + within).to(torch.int32)
        frequencies, state["magnitude"] = _frequencies(case)
        # Turns per position as a 64-bit fraction: a position times it, modulo
        # one turn, is exact at any position.
        steps = (frequencies / (2 * math.pi) * 2.0 ** 62).round().to(torch.int64) << 2
        state["steps"] = steps.to(DEVICE)
        if own:
            from cxlsparse_b200.rotary import Rotary

            scaling = {"none": None, "linear": dict(type="linear", factor=4.0),
                       "ntk": dict(type="ntk", factor=4.0),
                       "yarn": dict(type="yarn", factor=4.0, original=4096)}[case["scaling"]]
            state["rotary"] = Rotary(dim, rotary_dim=case["rotary"], theta=10000.0,
                                     layout=case["layout"], scaling=scaling, device=DEVICE)
        return state
    old = _history(case)
    lengths = [o + n for o, n in zip(old, new)]
    written = old if case["op"] == "append" else lengths
    state.update(_cache(case, g, lengths, new, written))
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    state["starts"] = torch.tensor(old, dtype=torch.int32, device=DEVICE)
    state["offsets"] = _offsets(new)
    if case["op"] == "append":
        channel = torch.exp(0.5 * _normal(g, 2, kv, dim))
        if case["fused"]:
            kvs = (_normal(g, total, 2, kv, dim) * channel).to(dtype)
            state["k"], state["v"] = kvs[:, 0], kvs[:, 1]
        else:
            state["k"] = (_normal(g, total, kv, dim) * channel[0]).to(dtype)
            state["v"] = (_normal(g, total, kv, dim) * channel[1]).to(dtype)
    if case["op"] == "attend":
        state["q"] = _normal(g, total, case["heads"], dim, dtype=dtype)
        state["scale"] = dim ** -0.5
    if own:
        from cxlsparse_b200.quantized import QuantizedCache

        state["cache"] = QuantizedCache(codes=state["codes"], scales=state["scales"])
    return state


# -------------------------------------------------------------- one pass ---


def run(state):
    case = state["case"]
    if not own:
        return {"rotary": _rotary, "append": _append, "read": _read,
                "attend": _attend}[case["op"]](state, case)
    if case["op"] == "rotary":
        q, k = state["rotary"].apply(state["q"], state["k"], state["positions"],
                                     transpose=case["transpose"])
        return {"q": q, "k": k}
    cache = state["cache"]
    if case["op"] == "append":
        cache.append(state["k"], state["v"], state["table"], state["lengths"], state["offsets"],
                     max_tokens=state["max_tokens"])
        return {"codes": cache.codes, "scales": cache.scales}
    if case["op"] == "read":
        k, v = cache.read(state["table"], state["starts"], state["offsets"],
                          total=sum(_tokens(case)), max_tokens=state["max_tokens"],
                          dtype=TYPES[case["dtype"]])
        return {"k": k, "v": v}
    out, lse = cache.attend(state["q"], state["table"], state["lengths"], state["offsets"],
                            max_tokens=state["max_tokens"], causal=case["causal"],
                            window=case["window"], scale=state["scale"], return_lse=True)
    return {"out": out, "lse": lse}


# The plain forms, in fp32.


def _rotary(state, case):
    phase = state["positions"].long()[:, None] * state["steps"]      # modulo 2^64
    angle = (phase >> 40).float() * (2 * math.pi / 2 ** 24)
    cos = (angle.cos() * state["magnitude"])[:, None, :]
    sin = (angle.sin() * state["magnitude"])[:, None, :]
    if case["transpose"]:
        sin = -sin
    d = case["rotary"]

    def turn(x):
        out = x.float()
        if case["layout"] == "half":
            a, b = out[..., :d // 2], out[..., d // 2:d]
            pair = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        else:
            a, b = out[..., 0:d:2], out[..., 1:d:2]
            pair = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        return torch.cat((pair, out[..., d:]), -1).to(x.dtype)

    return {"q": turn(state["q"]), "k": turn(state["k"])}


def _append(state, case):
    page, top = case["page"], TOP[case["format"]]
    codes, scales, table = state["codes"], state["scales"], state["table"]
    lengths, starts, offsets = state["lengths"], state["starts"], state["offsets"]
    # Every page that may get new tokens, and those of them that do.
    reach = torch.arange(-(-state["max_tokens"] // page) + 1, device=lengths.device)
    block = starts[:, None] // page + reach
    user, at = torch.nonzero(block * page < lengths[:, None], as_tuple=True)
    block = block[user, at]
    pages = table[user, block].long()
    position = block[:, None] * page + torch.arange(page, device=lengths.device)
    old = position < starts[user, None]
    new = (position < lengths[user, None]) & ~old
    token = (offsets[user, None] + position - starts[user, None]).clamp(0, len(state["k"]) - 1)
    x = torch.stack((state["k"], state["v"]), 2).float()[token]  # [n, page, heads, 2, dim]
    x = x.permute(0, 2, 3, 1, 4)
    old, new = old[:, None, None, :, None], new[:, None, None, :, None]
    size = torch.where(new & x.isfinite(), x.abs(), 0.0).amax((-2, -1))
    scale = (size * (1 / top)).clamp(min=LEAST)
    before = torch.where(old.any(-2)[..., 0], scales[pages], 0.0)
    scale = torch.maximum(scale, before)
    ratio = (before / scale)[..., None, None]
    held = codes[pages]
    again = _to_codes(case, held.float() * ratio)
    fresh = _to_codes(case, x * (torch.ones_like(scale) / scale)[..., None, None])
    held, again, fresh = (t.view(torch.uint8) for t in (held, again, fresh))
    codes.view(torch.uint8)[pages] = torch.where(new, fresh, torch.where(old, again, held))
    scales[pages] = scale
    return {"codes": codes, "scales": scales}


def _gather(state, case, positions, known):
    """K and V [..., heads, 2, dim] of the tokens at `positions` [users, n]."""
    page = case["page"]
    user = torch.arange(len(positions), device=positions.device)[:, None]
    block = (positions // page).clamp(0, state["table"].shape[1] - 1)
    pages = state["table"][user, block].long().clamp(min=0)
    rows = state["codes"].view(torch.uint8)[pages, :, :, positions % page]
    values = rows.view(state["codes"].dtype).float() * state["scales"][pages][..., None]
    return torch.where(known[..., None, None, None], values, 0.0)


def _packed(state, total):
    """(sequence, index within it) of every packed row."""
    row = torch.arange(total, device=state["offsets"].device, dtype=torch.int32)
    user = torch.searchsorted(state["offsets"][1:].contiguous(), row, right=True)
    return user, row - state["offsets"][user]


def _read(state, case):
    total = sum(_tokens(case))
    user, at = _packed(state, total)
    position = state["starts"][user] + at
    pages = state["table"][user, position // case["page"]].long()
    rows = state["codes"].view(torch.uint8)[pages, :, :, position % case["page"]]
    values = rows.view(state["codes"].dtype).float() * state["scales"][pages][..., None]
    values = values.to(TYPES[case["dtype"]])
    return {"k": values[:, :, 0].contiguous(), "v": values[:, :, 1].contiguous()}


def _attend(state, case):
    q, lengths, starts = state["q"], state["lengths"], state["starts"]
    users, kv, dim, most = case["users"], case["kv_heads"], case["dim"], state["max_tokens"]
    total, heads = q.shape[:2]
    key = torch.arange(state["table"].shape[1] * case["page"], device=q.device)
    known = key < lengths[:, None]
    kvs = _gather(state, case, key.expand(users, -1), known)       # [users, keys, kv, 2, dim]
    k, v = kvs[:, :, :, 0].permute(0, 2, 3, 1), kvs[:, :, :, 1].transpose(1, 2)
    user, at = _packed(state, total)
    rows = torch.zeros(users, most, heads, dim, device=q.device)
    rows[user, at] = q.float()
    rows = rows.view(users, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    rows = rows.reshape(users, kv, heads // kv * most, dim)
    s = (rows @ k * state["scale"]).view(users, kv, heads // kv, most, -1)
    position = starts[:, None] + torch.arange(most, device=q.device)
    seen = known[:, None, :].expand(-1, most, -1)
    if case["causal"]:
        seen = seen & (key <= position[..., None])
    if case["window"]:
        seen = seen & (key > position[..., None] - case["window"])
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = s.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    out = (p.view(users, kv, -1, len(key)) @ v).view(users, kv, heads // kv, most, dim)
    out = torch.where(l > 0, out / l, 0.0)
    lse = (m + l.log())[..., 0]

    def pack(x):  # [users, kv, group, tokens, ...] -> [total, heads, ...]
        return x.flatten(1, 2).transpose(1, 2)[user, at]

    return {"out": pack(out).to(q.dtype), "lse": pack(lse)}


# ------------------------------------------------------------- in 64 bits ---


def _nearest(case, x):
    """Nearest value of the format, ties to even, in fp64."""
    if case["format"] == "int8":
        return x.nan_to_num(nan=0.0).round().clamp(-127, 127)
    _, e = torch.frexp(x)
    unit = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return (x / unit).round().mul(unit).clamp(-448, 448)


def exact(case, seed):
    if case["op"] == "attend" and _pairs(case) * case["heads"] * case["dim"] > 5e11:
        return None
    state = prepare(case, seed)
    if case["op"] == "rotary":
        frequencies, magnitude = _frequencies(case)
        angle = state["positions"].double()[:, None] * frequencies.to(DEVICE)
        if case["transpose"]:
            angle = -angle
        z = torch.polar(torch.full_like(angle, magnitude), angle)[:, None]
        d, found = case["rotary"], {}
        for name in ("q", "k"):
            x = state[name].double()
            y = x.clone()
            if case["layout"] == "half":
                w = torch.complex(x[..., :d // 2], x[..., d // 2:d]) * z
                y[..., :d // 2], y[..., d // 2:d] = w.real, w.imag
            else:
                w = torch.complex(x[..., 0:d:2], x[..., 1:d:2]) * z
                y[..., 0:d:2], y[..., 1:d:2] = w.real, w.imag
            found[name] = y
        return found
    page, table, new, old = case["page"], state["table"].tolist(), _tokens(case), _history(case)
    first = state["offsets"].tolist()
    held = state["codes"].double()                   # in units of the scale
    scales = state["scales"].double()
    if case["op"] == "append":
        for b, (n, o) in enumerate(zip(new, old)):
            for j in range(o // page, -(-(o + n) // page)):
                low, high = max(o, j * page), min(o + n, (j + 1) * page)
                rows = slice(first[b] + low - o, first[b] + high - o)
                fill, p = low - j * page, table[b][j]
                x = torch.stack((state["k"][rows], state["v"][rows]), 2).double()
                x = x.permute(1, 2, 0, 3)            # [heads, 2, tokens, dim]
                scale = (x.abs().amax((-2, -1)) / TOP[case["format"]]).clamp(min=LEAST)
                if fill:
                    scale = torch.maximum(scale, scales[p])
                    held[p, :, :, :fill] = _nearest(
                        case, held[p, :, :, :fill] * (scales[p] / scale)[..., None, None])
                held[p, :, :, fill:high - j * page] = _nearest(case, x / scale[..., None, None])
                scales[p] = scale
        return {"codes": held if case["format"] == "e4m3" else None, "scales": scales}
    values = held * scales[..., None, None]          # [pages, heads, 2, page, dim]

    def tokens(b, low, high):
        blocks = values[table[b][low // page:-(-high // page)]]
        flat = blocks.permute(1, 2, 0, 3, 4).flatten(2, 3)
        return flat[:, :, low % page:low % page + high - low]

    if case["op"] == "read":
        rows = [tokens(b, o, o + n) for b, (n, o) in enumerate(zip(new, old))]
        rows = torch.cat(rows, 2).permute(1, 2, 0, 3)
        return {"k": rows[0], "v": rows[1]}
    group = case["heads"] // case["kv_heads"]
    outs, lses = [], []
    for b, (n, o) in enumerate(zip(new, old)):
        k, v = tokens(b, 0, o + n).unbind(1)         # [kv heads, keys, dim]
        q = state["q"][first[b]:first[b + 1]].double().view(n, -1, group, case["dim"])
        position = torch.arange(o, o + n, device=DEVICE)[:, None]
        key = torch.arange(o + n, device=DEVICE)
        hidden = torch.zeros(n, o + n, dtype=torch.bool, device=DEVICE)
        if case["causal"]:
            hidden |= key > position
        if case["window"]:
            hidden |= key <= position - case["window"]
        out, lse = [], []
        for h in range(case["kv_heads"]):
            s = torch.einsum("ngd,kd->ngk", q[:, h], k[h]) * state["scale"]
            s = s.masked_fill(hidden[:, None], -math.inf)
            m = torch.logsumexp(s, -1)
            out.append(torch.einsum("ngk,kd->ngd", torch.exp(s - m[..., None]), v[h]))
            lse.append(m)
        outs.append(torch.cat(out, 1))
        lses.append(torch.cat(lse, 1))
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
