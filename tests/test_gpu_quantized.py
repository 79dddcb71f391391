"""The dense 8-bit cache on the device against plain fp64 forms."""

import math

import pytest
import torch

from cache8_case import CODE, TOP, UNIT, attend, nearest, offsets_of, paged, tokens_of
from cxlsparse_b200 import CxsError
from cxlsparse_b200.quantized import QuantizedCache

pytestmark = pytest.mark.gpu

FORMATS = ["e4m3", "int8"]
LEAST = 2.0 ** -64


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def raw(t):
    return t.view(torch.uint8)


# ----------------------------------------------------------------- append ---


def appended(codes, scales, table, lengths, new, k, v, format):
    """The append's own fp32 sequence, page by page (on the device, elementary
    operations): bit for bit what the kernel writes."""
    codes, scales = codes.clone(), scales.clone()
    page, top = codes.shape[3], TOP[format]
    at = 0
    for b, (length, n) in enumerate(zip(lengths, new)):
        start = length - n
        for j in range(start // page, -(-length // page) if n else 0):
            low, high = max(start, j * page), min(length, (j + 1) * page)
            fill, stop, p = low - j * page, high - j * page, int(table[b, j])
            x = torch.stack((k, v), 2).float()[at + low - start:at + high - start]
            x = x.permute(1, 2, 0, 3)                               # [heads, 2, n, dim]
            size = torch.where(x.isfinite(), x.abs(), 0.0).amax((-2, -1))
            scale = (size * (1 / top)).clamp(min=LEAST)
            held = raw(codes)[p]
            if fill:
                before = scales[p].clone()
                scale = torch.maximum(scale, before)
                old = held[:, :, :fill].contiguous().view(CODE[format]).float()
                old = old * (before / scale)[..., None, None]
                held[:, :, :fill] = encode(old, format)
            inverse = torch.ones_like(scale) / scale
            held[:, :, fill:stop] = encode(x * inverse[..., None, None], format)
            raw(codes)[p] = held
            scales[p] = scale
        at += n
    return codes, scales


def encode(x, format):
    x = x.clamp(-TOP[format], TOP[format])
    if format == "e4m3":
        return raw(x.to(torch.float8_e4m3fn))
    return raw(x.nan_to_num(nan=0.0).round().to(torch.int8))


APPENDS = [
    # lengths before, new tokens
    ([0], [1]), ([63], [1]), ([64], [1]), ([64], [2]), ([5], [300]), ([0], [64]),
    ([0, 1, 15, 16, 17, 130], [0, 1, 2, 16, 33, 129]), ([100, 0, 0, 31], [1, 0, 128, 1]),
]


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim,page", [(64, 64), (64, 16), (128, 32), (128, 64)])
@pytest.mark.parametrize("before,new", APPENDS)
def test_append_is_the_fp32_sequence(cuda, format, dtype, dim, page, before, new):
    heads = 3
    lengths = [o + n for o, n in zip(before, new)]
    codes, scales, table = paged(before, kv_heads=heads, dim=dim, page_size=page, format=format)
    grown = torch.full((len(new), max(-(-n // page) for n in lengths) + 1), -1,
                       dtype=torch.int32, device="cuda")
    grown[:, :table.shape[1]] = table
    fresh = len(codes)                       # new pages behind the old ones
    for b, (o, n) in enumerate(zip(before, lengths)):
        for j in range(-(-o // page), -(-n // page)):
            grown[b, j] = fresh
            fresh += 1
    extra = fresh - len(codes)
    codes = torch.cat((raw(codes), raw(codes).new_full((extra, *codes.shape[1:]), 0xFF)))
    codes = codes.view(CODE[format])
    scales = torch.cat((scales, scales.new_full((extra, *scales.shape[1:]), math.nan)))
    g = torch.Generator(device="cuda").manual_seed(3)
    total = sum(new)
    kv = torch.randn(total, 2, heads, dim, generator=g, device="cuda")
    kv = (kv * torch.exp(torch.randn(total, 2, heads, 1, generator=g, device="cuda"))).to(dtype)
    k, v = kv[:, 0], kv[:, 1]                # strided views
    expect = appended(codes, scales, grown, lengths, new, k, v, format)
    cache = QuantizedCache(codes=codes.clone(), scales=scales.clone())
    cache.append(k, v, grown, ints(lengths), offsets_of(new), max_tokens=max(new))
    cache.check()
    assert torch.equal(raw(cache.codes), raw(expect[0]))
    torch.testing.assert_close(cache.scales, expect[1], rtol=0, atol=0, equal_nan=True)
    # Without the host's bound on the tokens of one user: the same.
    again = QuantizedCache(codes=codes.clone(), scales=scales.clone())
    again.append(k.contiguous(), v.contiguous(), grown, ints(lengths), offsets_of(new))
    assert torch.equal(raw(again.codes), raw(expect[0]))
    # Against the definition in fp64: every new value is within half a code
    # step of the input (2^-22: the fp32 reciprocal, product and scale).
    at = 0
    for b, (length, n) in enumerate(zip(lengths, new)):
        if n:
            got = tokens_of(cache.codes, cache.scales, grown, b, length - n, length)
            ids = grown[b, (torch.arange(length - n, length, device="cuda") // page)].long()
            for part, x in enumerate((k, v)):
                x = x[at:at + n].double().transpose(0, 1)
                s = cache.scales[ids, :, part].double().T[..., None]
                unit = x / s
                step = torch.ones_like(unit) if format == "int8" else torch.ldexp(
                    torch.ones_like(unit), (torch.frexp(unit)[1] - 4).clamp(min=-9))
                bound = (0.5 * step + 2.0 ** -22 * unit.abs()) * s
                assert ((got[part] - x).abs() <= bound).all()
        at += n


@pytest.mark.parametrize("format", FORMATS)
def test_append_one_token_at_a_time_follows_the_same_sequence(cuda, format):
    """Token by token: pages whose scale grows as larger tokens come."""
    heads, dim, page = 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.zeros(4, heads, 2, page, dim, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(4, heads, 2, device="cuda")
    table = ints([[2, 0], [1, 3]])
    cache = QuantizedCache(codes=codes.view(CODE[format]).clone(), scales=scales.clone())
    expect = (codes.view(CODE[format]), scales)
    for t in range(25):
        k = torch.randn(2, heads, dim, generator=g, device="cuda") * (1 + t % 7)
        v = torch.randn(2, heads, dim, generator=g, device="cuda") / (1 + t % 5)
        lengths = [t + 1, t + 1]
        cache.append(k, v, table, ints(lengths))
        expect = appended(*expect, table, lengths, [1, 1], k, v, format)
    cache.check()
    assert torch.equal(raw(cache.codes), raw(expect[0]))
    assert torch.equal(cache.scales, expect[1])


@pytest.mark.parametrize("format", FORMATS)
def test_append_zeros_infinities_and_nan(cuda, format):
    heads, dim, page = 1, 64, 16
    cache = QuantizedCache(3, heads, dim, page_size=page, format=format)
    table = ints([[0, 1, 2]])
    k = torch.zeros(40, heads, dim, device="cuda")
    v = torch.randn(40, heads, dim, device="cuda")
    k[20] = 1e-30                             # below the smallest scale
    k[35, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 2.0])
    cache.append(k, v, table, ints([40]), ints([0, 40]))
    cache.check()
    values = cache.codes.float()
    assert (values[0, 0, 0] == 0).all() and cache.scales[0, 0, 0] == LEAST
    assert cache.scales[1, 0, 0] == LEAST and (values[1, 0, 0] == 0).all()
    top = TOP[format]
    assert cache.scales[2, 0, 0] == torch.tensor(2.0) * torch.tensor(1 / top)
    row = values[2, 0, 0, 3]
    assert row[0] == top and row[1] == -top and row[3] == top
    assert row[2].isnan() if format == "e4m3" else row[2] == 0


def test_append_keeps_other_pages_and_reports_what_is_out_of_range(cuda):
    heads, dim, page = 2, 64, 16
    cache = QuantizedCache(4, heads, dim, page_size=page, format="int8")
    raw(cache.codes).fill_(7)
    cache.scales.fill_(0.5)
    k = torch.randn(6, heads, dim, device="cuda")
    # A page id past the cache and one below zero: skipped, the rest written.
    cache.append(k, k, ints([[9, 1], [-1, 2], [3, 0]]), ints([2, 2, 2]), ints([0, 2, 4, 6]))
    with pytest.raises(CxsError, match="page id"):
        cache.check()
    cache.check()                             # reported once
    assert (raw(cache.codes)[:3] == 7).all() and (cache.scales[:3] == 0.5).all()
    assert (raw(cache.codes)[3, :, :, 2:] == 7).all()
    assert not (raw(cache.codes)[3, :, :, :2] == 7).all()
    # Lengths past the table, rows past the packed tokens, fewer tokens than rows.
    for lengths, offsets in (([33], [0, 2]), ([8], [0, 9]), ([1], [0, 4]), ([4], [3, 1])):
        cache.append(k, k, ints([[0, 1]]), ints(lengths), ints(offsets))
        with pytest.raises(CxsError, match="lengths or offsets"):
            cache.check()
    cache.append(k, k, ints([[0, 1]]), ints([6]), ints([0, 6]), max_tokens=3)
    with pytest.raises(CxsError, match="lengths or offsets"):
        cache.check()


# ------------------------------------------------------------------- read ---


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim,page", [(64, 64), (64, 16), (128, 32)])
@pytest.mark.parametrize("lengths,starts,new", [
    ([1], [0], [1]), ([200], [0], [200]), ([200], [63], [66]), ([200], [199], [1]),
    ([130, 0, 17, 64, 500], [3, 0, 16, 0, 251], [127, 0, 1, 64, 200]),
])
def test_read_is_code_times_scale_rounded_once(cuda, format, dtype, dim, page, lengths, starts,
                                               new):
    codes, scales, table = paged(lengths, kv_heads=3, dim=dim, page_size=page, format=format)
    cache = QuantizedCache(codes=codes, scales=scales)
    k, v = cache.read(table, ints(starts), offsets_of(new), total=sum(new), dtype=dtype,
                      max_tokens=max(new))
    cache.check()
    at = 0
    for b, (start, n) in enumerate(zip(starts, new)):
        for got, want in zip((k, v), tokens_of(codes, scales, table, b, start, start + n)):
            # The fp32 product of a code and a scale, then one rounding.
            assert torch.equal(got[at:at + n], want.transpose(0, 1).float().to(dtype))
        at += n


def test_read_out_of_range_gives_zeros_and_an_error(cuda):
    codes, scales, table = paged([64], kv_heads=2, dim=64, page_size=16, format="int8")
    cache = QuantizedCache(codes=codes, scales=scales)
    broken = table.clone()
    broken[0, 1] = len(codes)
    k, v = cache.read(broken, ints([0]), ints([0, 64]), total=64, dtype=torch.float32)
    with pytest.raises(CxsError, match="page id"):
        cache.check()
    assert (k[16:32] == 0).all() and (v[16:32] == 0).all()
    whole = cache.read(table, ints([0]), ints([0, 64]), total=64, dtype=torch.float32)
    assert torch.equal(k[32:], whole[0][32:]) and torch.equal(v[:16], whole[1][:16])
    for starts in (-5, 60):
        k, v = cache.read(table, ints([starts]), ints([0, 20]), total=20, dtype=torch.float32)
        with pytest.raises(CxsError, match="lengths or offsets"):
            cache.check()
        low, high = max(0, -starts), min(20, 64 - starts)
        assert torch.equal(k[low:high], whole[0][starts + low:starts + high])
        assert (k[:low] == 0).all() and (v[high:] == 0).all()


# ----------------------------------------------------------------- attend ---


def check_attend(lengths, new, *, heads, kv_heads, dim, page, format, dtype, causal=True,
                 window=0, seed=0, gain=1.0, max_tokens=True, spread=1.0):
    codes, scales, table = paged(lengths, kv_heads=kv_heads, dim=dim, page_size=page,
                                 format=format, seed=seed, spread=spread)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = (gain * torch.randn(sum(new), heads, dim, generator=g, device="cuda")).to(dtype)
    cache = QuantizedCache(codes=codes, scales=scales)
    out, lse = cache.attend(q, table, ints(lengths), offsets_of(new),
                            max_tokens=max(new) if max_tokens else None, causal=causal,
                            window=window, return_lse=True)
    cache.check()
    want, want_lse, tol, tol_lse = attend(q, codes, scales, table, lengths, new, causal=causal,
                                          window=window, scale=dim ** -0.5)
    assert out.dtype == dtype and out.shape == q.shape
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (out[empty] == 0).all()
    assert ((out.double() - want).abs() <= tol).all(), ((out.double() - want).abs() / tol).max()
    off = (lse.double() - want_lse).abs()[~empty]
    assert (off <= tol_lse[~empty]).all()
    return cache, q, table, out, lse


LENGTHS = [
    [1], [2], [15], [16], [17], [63], [64], [65], [127], [1000], [4097],
    [0], [0, 5, 0], [1, 64, 129, 0, 700, 33, 2, 255],
]


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dim,page", [(64, 64), (64, 16), (128, 64), (128, 32)])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_attend_one_token_each(cuda, format, dim, page, lengths):
    check_attend(lengths, [1] * len(lengths), heads=32, kv_heads=2, dim=dim, page=page,
                 format=format, dtype=torch.bfloat16)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (12, 4), (16, 1), (20, 1), (40, 1),
                                            (64, 2), (71, 1)])
@pytest.mark.parametrize("new", [1, 3, 8])
def test_attend_head_layouts(cuda, heads, kv_heads, new):
    for format, dim, dtype in (("e4m3", 64, torch.float16), ("int8", 128, torch.bfloat16)):
        check_attend([300, 77], [new, new], heads=heads, kv_heads=kv_heads, dim=dim, page=32,
                     format=format, dtype=dtype)


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 100),
                                           (False, 65), (True, 5000)])
@pytest.mark.parametrize("lengths,new", [
    ([300], [40]), ([129, 64, 1000], [129, 3, 70]), ([5], [17]), ([0, 200], [4, 150]),
    ([700], [300]),
], ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_suffixes_and_masks(cuda, format, causal, window, lengths, new, dim):
    """Suffixes and prefills; more rows than tokens leaves rows that see nothing."""
    check_attend(lengths, new, heads=16, kv_heads=2, dim=dim, page=64, format=format,
                 dtype=torch.bfloat16, causal=causal, window=window)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_attend_long_ragged_batch(cuda, dim, page):
    lengths = [9000, 1, 0, 20011, 333, 64, 4096, 12345]
    for new in ([1] * 8, [2, 1, 3, 4, 1, 5, 0, 16], [40, 1, 0, 200, 90, 64, 1, 130]):
        check_attend(lengths, new, heads=8, kv_heads=2, dim=dim, page=page, format="int8",
                     dtype=torch.float16)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dtype,gain", [(torch.bfloat16, 1e-3), (torch.bfloat16, 20.0),
                                        (torch.float16, 20.0), (torch.float16, 1e-3)])
def test_attend_flat_and_peaked_scores_and_wide_scales(cuda, new, dtype, gain):
    """Scores near zero and in the hundreds; page scales over ten orders."""
    check_attend([1500, 90], [new, new], heads=16, kv_heads=1, dim=64, page=16, format="e4m3",
                 dtype=dtype, gain=gain)
    codes, scales, table = paged([600], kv_heads=1, dim=64, page_size=16, format="int8")
    g = torch.Generator(device="cuda").manual_seed(5)
    scales[..., 1] *= 10.0 ** (10 * torch.rand(scales[..., 1].shape, generator=g,
                                               device="cuda") - 8)
    q = torch.randn(new, 16, 64, generator=g, device="cuda").to(dtype)
    cache = QuantizedCache(codes=codes, scales=scales)
    out = cache.attend(q, table, ints([600]), ints([0, new]), max_tokens=new)
    want, _, tol, _ = attend(q, codes, scales, table, [600], [new], causal=True, window=0,
                             scale=64 ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("new", [1, 2, 50])
def test_attend_strided_unaligned_queries_other_stream_and_repeats(cuda, new):
    lengths, counts = [800, 333], [new, new]
    codes, scales, table = paged(lengths, kv_heads=2, dim=64, page_size=64, format="e4m3")
    cache = QuantizedCache(codes=codes, scales=scales)
    args = (table, ints(lengths), offsets_of(counts))
    fused = torch.randn(2 * new, 8 * 64 + 2 * 2 * 64 + 24, device="cuda").bfloat16()
    q = fused[:, :512].view(2 * new, 8, 64)
    plain = cache.attend(q.contiguous(), *args, max_tokens=new)
    assert torch.equal(cache.attend(q, *args, max_tokens=new), plain)
    shifted = torch.empty(2 * new * 8 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:]
    shifted = shifted.view(2 * new, 8, 64).copy_(q)                     # 2-byte alignment
    assert torch.equal(cache.attend(shifted, *args, max_tokens=new), plain)
    padded = torch.zeros(2, table.shape[1] + 5, dtype=torch.int32, device="cuda") - 1
    padded[:, :table.shape[1]] = table
    assert torch.equal(cache.attend(q, padded[:, :table.shape[1]], *args[1:], max_tokens=new),
                       plain)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [cache.attend(q, *args, max_tokens=new) for _ in range(20)]
    mine = [cache.attend(q, *args, max_tokens=new) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, plain) for x in others + mine)            # same bits every time


def test_attend_does_not_depend_on_unused_bytes(cuda):
    lengths = [100, 17]
    for new in ([1, 1], [80, 10]):
        codes, scales, table = paged(lengths, kv_heads=1, dim=64, page_size=64, format="e4m3")
        args = (ints(lengths), offsets_of(new))
        q = torch.randn(sum(new), 4, 64, device="cuda").bfloat16()
        first = QuantizedCache(codes=codes, scales=scales).attend(q, table, *args)
        clean = raw(codes).clone()
        clean[clean == 0xFF] = 0
        clean = clean.view(codes.dtype)
        second = QuantizedCache(codes=clean, scales=scales.nan_to_num()).attend(q, table, *args)
        assert torch.equal(first, second)


@pytest.mark.parametrize("new", [1, 70])
def test_attend_nan_of_a_visible_token_stays_in_its_rows(cuda, new):
    """A NaN key reaches the rows that see it and no other row."""
    codes, scales, table = paged([200, 200], kv_heads=1, dim=64, page_size=64, format="e4m3")
    raw(codes)[table[1, 3], 0, 0, 5] = 0x7F                # user 1's token 197
    cache = QuantizedCache(codes=codes, scales=scales)
    q = torch.randn(2 * new, 16, 64, device="cuda").bfloat16()
    out, lse = cache.attend(q, table, ints([200, 200]), offsets_of([new, new]),
                            return_lse=True)
    assert not out[:new].isnan().any()
    position = torch.arange(200 - new, 200, device="cuda")
    assert torch.equal(out[new:].isnan().all(-1).all(-1), position >= 197)
    assert not out[new:][position < 197].isnan().any()
    assert torch.equal(lse[new:].isnan().all(-1), position >= 197)


@pytest.mark.parametrize("new", [1, 70])
def test_attend_skips_pages_out_of_range(cuda, new):
    codes, scales, table = paged([256], kv_heads=2, dim=64, page_size=16, format="int8")
    cache = QuantizedCache(codes=codes, scales=scales)
    q = torch.randn(new, 8, 64, device="cuda").bfloat16()
    whole = cache.attend(q, table, ints([128]), ints([0, new]), causal=False)
    broken = table.clone()
    broken[0, 8:] = torch.tensor([-1, len(codes), -7, 1 << 30] * 2, device="cuda")
    out = cache.attend(q, broken, ints([256]), ints([0, new]), causal=False)
    with pytest.raises(CxsError, match="page id"):
        cache.check()
    torch.testing.assert_close(out.float(), whole.float(), rtol=2 ** -7, atol=1e-5)
    # More tokens than the table holds: cut, with the error bit.
    cut = cache.attend(q, table[:, :8], ints([1000]), ints([0, new]), causal=False)
    with pytest.raises(CxsError, match="lengths or offsets"):
        cache.check()
    torch.testing.assert_close(cut.float(), whole.float(), rtol=2 ** -7, atol=1e-5)
    # Rows that belong to no user are empty.
    q3 = torch.cat((q, q))
    out, lse = cache.attend(q3, table, ints([128]), ints([0, new]), causal=False,
                            return_lse=True)
    cache.check()
    assert (out[new:] == 0).all() and (lse[new:] == -math.inf).all()
    assert torch.equal(out[:new], whole)


@pytest.mark.parametrize("dim", [64, 128])
def test_attend_full_and_half_items_in_turn(cuda, dim):
    """Items whose second 128 rows are there, partly there and missing, one after
    the other and in every order, over few and many key tiles: the groups of
    rows pass each other's tiles."""
    g = torch.Generator().manual_seed(0)
    for trial in range(6):
        users = 24
        lengths = torch.randint(1, 1500, (users,), generator=g).tolist()
        new = [int(torch.randint(1, 130, (1,), generator=g)) if i % 2 == trial % 2
               else (1, 30, 64, 65, 127, 128)[i // 2 % 6] for i in range(users)]
        for _ in range(3):
            check_attend(lengths, new, heads=4, kv_heads=2, dim=dim, page=32, format="e4m3",
                         dtype=torch.float16, seed=trial)


@pytest.mark.parametrize("new", [1, 300])
@pytest.mark.parametrize("scale", [-0.125, 0.0, 1.0])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_any_scale_on_the_scores(cuda, new, scale, dim):
    lengths = [700, 301]
    codes, scales, table = paged(lengths, kv_heads=2, dim=dim, page_size=32, format="int8")
    q = 0.2 * torch.randn(2 * new, 8, dim, device="cuda").bfloat16()
    out, lse = QuantizedCache(codes=codes, scales=scales).attend(
        q, table, ints(lengths), offsets_of([new, new]), max_tokens=new, scale=scale,
        return_lse=True)
    want, want_lse, tol, tol_lse = attend(q, codes, scales, table, lengths, [new, new],
                                          causal=True, window=0, scale=scale)
    assert ((out.double() - want).abs() <= tol).all()
    assert ((lse.double() - want_lse).abs() <= tol_lse).all()


@pytest.mark.parametrize("dim,new", [(64, 1), (128, 1), (64, 9), (128, 33)])
def test_attend_one_long_user_is_split_over_the_gpu(cuda, dim, new):
    """100,001 tokens of one user: every SM holds a part of the same item."""
    check_attend([100001], [new], heads=8, kv_heads=1, dim=dim, page=64, format="e4m3",
                 dtype=torch.bfloat16)


@pytest.mark.parametrize("new", [1, 20])
def test_attend_more_users_than_one_launch_holds(cuda, new):
    """4,500 users of 0 to 40 tokens: three launches of at most 2048 users, many
    items for every worker."""
    lengths = [(i * 37) % 41 for i in range(4500)]
    counts = [new if i % 3 else 0 for i in range(4500)]
    check_attend(lengths, counts, heads=8, kv_heads=1, dim=64, page=16, format="int8",
                 dtype=torch.float16)
    if new == 1:
        codes, scales, table = paged(lengths, kv_heads=1, dim=64, page_size=16, format="int8")
        q = torch.randn(4500, 8, 64, device="cuda").half()
        cache = QuantizedCache(codes=codes, scales=scales)
        packed = cache.attend(q, table, ints(lengths), offsets_of([1] * 4500), max_tokens=1)
        assert torch.equal(cache.attend(q, table, ints(lengths)), packed)


def test_append_unaligned_rows(cuda):
    """Rows that start 2 bytes past a 16-byte boundary, of uneven strides."""
    rows = torch.randn(70, 2 * 2 * 64 + 9, device="cuda").bfloat16()
    k, v = (rows[:, 1 + 128 * i:129 + 128 * i].view(70, 2, 64) for i in range(2))
    table = ints([[1, 0, 2, 3, 4]])
    first, second = (QuantizedCache(5, 2, 64, page_size=16, format="e4m3") for _ in range(2))
    first.append(k, v, table, ints([70]), ints([0, 70]))
    second.append(k.contiguous(), v.contiguous(), table, ints([70]), ints([0, 70]))
    first.check()
    assert torch.equal(raw(first.codes), raw(second.codes))
    assert torch.equal(first.scales, second.scales)


def test_attend_of_nothing(cuda):
    cache = QuantizedCache(2, 1, 64)
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    out, lse = cache.attend(q, table, ints([3, 0]), ints([0, 0, 0]), return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    k = torch.empty(0, 1, 64, dtype=torch.bfloat16, device="cuda")
    cache.append(k, k, table, ints([3, 0]), ints([0, 0, 0]))
    k, v = cache.read(table, ints([0, 0]), ints([0, 0, 0]), total=0)
    assert k.shape == v.shape == (0, 1, 64)


def test_append_then_attend_in_a_graph(cuda):
    """A captured step: append, attend; replayed with new inputs in place."""
    heads, kv, dim, page = 8, 2, 64, 16
    cache = QuantizedCache(8, kv, dim, page_size=page, format="e4m3")
    table, lengths = ints([[0, 2, 4], [1, 3, 5]]), ints([1, 20])
    raw(cache.codes).zero_()
    cache.scales.fill_(2.0 ** -64)
    q = torch.zeros(2, heads, dim, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.zeros(2, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(k, v, table, lengths)
        out = cache.attend(q, table, lengths)
    twin = QuantizedCache(codes=cache.codes.clone(), scales=cache.scales.clone())
    g = torch.Generator(device="cuda").manual_seed(0)
    for step in range(12):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        graph.replay()
        twin.append(k, v, table, lengths)
        assert torch.equal(twin.attend(q, table, lengths), out)
        assert torch.equal(raw(twin.codes), raw(cache.codes))
        lengths += 1
    cache.check()


def test_large_offsets_pass_32_bits(cuda):
    """Pages whose bytes lie past 2^32 (a 5 GB cache)."""
    heads, dim, page = 8, 128, 64
    pages = 5 * 2 ** 30 // (heads * 2 * page * dim)
    codes = torch.empty(pages, heads, 2, page, dim, dtype=torch.int8, device="cuda")
    scales = torch.empty(pages, heads, 2, device="cuda")
    cache = QuantizedCache(codes=codes, scales=scales)
    table = ints([[pages - 1, 3, pages - 2, 0]])
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(200, heads, dim, generator=g, device="cuda").half() for _ in range(2))
    cache.append(k, v, table, ints([200]), ints([0, 200]))
    back_k, back_v = cache.read(table, ints([0]), ints([0, 200]), total=200, dtype=torch.float16)
    cache.check()
    step = k.abs().amax().float() / 127
    assert ((back_k.float() - k.float()).abs() <= 0.51 * step).all()
    for new in (1, 100):
        q = torch.randn(new, 16, dim, generator=g, device="cuda").half()
        out = cache.attend(q, table, ints([200]), ints([0, new]))
        want, _, tol, _ = attend(q, codes, scales, table, [200], [new], causal=True, window=0,
                                 scale=dim ** -0.5)
        assert ((out.double() - want).abs() <= tol).all()
    cache.check()


def test_nearest_matches_the_format(cuda):
    """The tests' own rounding is torch's conversion to the format."""
    x = torch.randn(100000, device="cuda") * 100
    assert torch.equal(nearest(x.double(), "e4m3").float(),
                       x.clamp(-448, 448).to(torch.float8_e4m3fn).float())
    assert all(u == torch.finfo(t).eps / 2 for t, u in UNIT.items())
