"""Cases of the dense 8-bit cache and their plain form in fp64.

Unused bytes (slots past a user's length, pages that no table row uses) hold
NaN codes, -1 and NaN scales: nothing of them may reach a result.
"""

import math

import torch

TOP = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def nearest(x, format):
    """Nearest code values to x (fp64), ties to even, saturated."""
    if format == "int8":
        return x.nan_to_num(nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127)
    x = x.clamp(-448, 448)
    _, e = torch.frexp(x)
    unit = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return (x / unit).round().mul(unit)


def paged(lengths, *, kv_heads, dim, page_size, format, seed=0, device="cuda", spare=2,
          spread=1.0):
    """(codes, scales, table): a cache holding lengths[b] random tokens of each
    user in shuffled pages. Codes use the whole range of the format; scales
    differ between pages by factors of about exp(spread)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page_size) for n in lengths]
    pages, width = sum(need) + spare, max(need + [1])
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    values = torch.randn(pages, kv_heads, 2, page_size, dim, generator=g, dtype=torch.float64)
    scales = torch.exp(spread * torch.randn(pages, kv_heads, 2, generator=g)) \
        * values.abs().amax((-2, -1)).float() / TOP[format]
    codes = nearest(values / (values.abs().amax((-2, -1), keepdim=True) / TOP[format]), format)
    codes = codes.to(CODE[format]).view(torch.uint8)
    hole = torch.ones(pages, page_size, dtype=torch.bool)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        for j in range(n):
            hole[table[b, j], :max(0, lengths[b] - j * page_size)] = False
        at += n
    codes[hole[:, None, None].expand(-1, kv_heads, 2, -1)] = 0xFF if format == "e4m3" else 0x80
    scales[hole.all(1)] = math.nan
    return codes.view(CODE[format]).to(device), scales.to(device), table.to(device)


def tokens_of(codes, scales, table, b, low, high):
    """fp64 (k, v) [kv_heads, high - low, dim] of user b's tokens low .. high - 1."""
    page_size = codes.shape[3]
    if high <= low:
        empty = torch.zeros(codes.shape[1], 0, codes.shape[4], dtype=torch.float64,
                            device=codes.device)
        return empty, empty
    ids = table[b, low // page_size:-(-high // page_size)].long()
    held = codes.view(torch.uint8)[ids].view(codes.dtype).double()
    values = held * scales[ids].double()[..., None, None]
    flat = values.permute(1, 2, 0, 3, 4).flatten(2, 3)
    flat = flat[:, :, low % page_size:low % page_size + high - low]
    return flat[:, 0], flat[:, 1]


def attend(q, codes, scales, table, lengths, new, *, causal, window, scale):
    """(out, lse, tolerance of out, tolerance of lse) in fp64 of packed queries.

    Tolerances, per element: scores are fp32 dot products (of at most 128
    terms: 2^-17 of the sum of magnitudes), probabilities are rounded to 11
    bits (2^-11 of the sum of p |v|, doubled for the exponential and the
    running sums; 2^-25 of the largest value where they underflow), and out is
    rounded to its type.
    """
    heads, kv = q.shape[1], codes.shape[1]
    outs, lses, tol_o, tol_l = [], [], [], []
    at = 0
    for b, (length, n) in enumerate(zip(lengths, new)):
        k, v = tokens_of(codes, scales, table, b, 0, length)
        rows = q[at:at + n].double().view(n, kv, heads // kv, q.shape[2])
        at += n
        position = torch.arange(length - n, length, device=q.device)[:, None]
        key = torch.arange(length, device=q.device)
        seen = torch.ones(n, length, dtype=torch.bool, device=q.device)
        if causal:
            seen &= key <= position
        if window:
            seen &= key > position - window
        s = torch.einsum("nhgd,hkd->nhgk", rows, k) * scale
        size = torch.einsum("nhgd,hkd->nhgk", rows.abs(), k.abs()) * abs(scale)
        s = s.masked_fill(~seen[:, None, None], -math.inf)
        size = size.masked_fill(~seen[:, None, None], 0.0)
        size = size.amax(-1) if length else size.new_zeros(size.shape[:-1])
        lse = torch.logsumexp(s, -1) if length else s.new_full(s.shape[:-1], -math.inf)
        p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
        out = torch.einsum("nhgk,hkd->nhgd", p, v)
        spread = torch.einsum("nhgk,hkd->nhgd", p, v.abs())
        most = v.abs().amax() if length else 0.0
        delta = 2.0 ** -17 * size
        tol = UNIT[q.dtype] * out.abs() + spread * (2.0 ** -10 + 2 * delta)[..., None] \
            + length * 2.0 ** -25 * most + 1e-7
        outs.append(out.flatten(1, 2))
        lses.append(lse.flatten(1, 2))
        tol_o.append(tol.flatten(1, 2))
        tol_l.append((delta + 4e-6 + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0)).flatten(1, 2))
    return tuple(torch.cat(x) for x in (outs, lses, tol_o, tol_l))


def offsets_of(new, device="cuda"):
    return torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32,
                        device=device)
