"""The 8-bit cache's results in norm, row by row: tolerances that neither the
length of a history nor its largest value widens.

The relative error of a row of out in norm: probabilities rounded to 11 bits,
independent from key to key (2^-11 / sqrt 3), out rounded to fp16 (the same)
and scores from fp32 sums (below 2^-13) make 1e-3; doubled for a row's luck.
Where out lies below 2^-14, its fp16 values are 2^-24 apart.
"""

import math

import pytest
import torch

from cache8_case import CODE, attend, offsets_of, paged, tokens_of
from cxlsparse_b200.quantized import QuantizedCache
from test_gpu_quantized import appended, raw

pytestmark = pytest.mark.gpu

LIMIT = 2e-3


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def check(lengths, new, *, heads, kv_heads, dim, page, format, spread=1.0, decades=0.0, gain=1.0,
          causal=True, window=0, seed=0):
    codes, scales, table = paged(lengths, kv_heads=kv_heads, dim=dim, page_size=page,
                                 format=format, spread=spread, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 7)
    if decades:
        scales[..., 1] *= 10.0 ** (decades * (torch.rand(scales[..., 1].shape, generator=g,
                                                         device="cuda") - 1))
    # Out of a long history is small: away from fp16's subnormals.
    scales[..., 1] *= 64.0
    q = (gain * torch.randn(sum(new), heads, dim, generator=g, device="cuda")).half()
    cache = QuantizedCache(codes=codes, scales=scales)
    out, lse = cache.attend(q, table, ints(lengths), offsets_of(new), max_tokens=max(new),
                            causal=causal, window=window, return_lse=True)
    cache.check()
    want, want_lse, _, tol_lse = attend(q, codes, scales, table, lengths, new, causal=causal,
                                        window=window, scale=dim ** -0.5)
    some = want_lse > -math.inf
    off = (out.double() - want)[some].norm(dim=-1)
    assert (off <= LIMIT * want[some].norm(dim=-1) + dim ** 0.5 * 2.0 ** -25).all()
    assert ((lse.double() - want_lse).abs() <= tol_lse)[some].all()


@pytest.mark.parametrize("format", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,new", [(64, 1), (128, 1), (64, 9), (128, 33)])
def test_one_long_user_joined_over_the_gpu(cuda, dim, new, format):
    check([100001], [new], heads=8, kv_heads=1, dim=dim, page=64, format=format)


@pytest.mark.parametrize("format", ["e4m3", "int8"])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_scales_over_ten_decades(cuda, new, dim, format):
    """out is that of the pages with the largest V scales; lse counts all."""
    check([600, 4000], [new, new], heads=16, kv_heads=1, dim=dim, page=16, format=format,
          decades=10.0)


@pytest.mark.parametrize("dim,page", [(64, 16), (64, 64), (128, 16), (128, 32), (128, 64)])
@pytest.mark.parametrize("new", [[1] * 8, [2, 1, 3, 4, 1, 5, 0, 16], [40, 1, 0, 200, 90, 64, 1, 130]],
                         ids=str)
@pytest.mark.parametrize("gain", [0.01, 1.0, 3.0])
def test_ragged_batches(cuda, dim, page, new, gain):
    check([9000, 1, 0, 20011, 333, 64, 4096, 12345], new, heads=8, kv_heads=2, dim=dim, page=page,
          format="e4m3" if page == 16 else "int8", gain=gain)


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 700), (False, 0), (False, 65)])
@pytest.mark.parametrize("new", [1, 7, 150])
def test_masks_at_128_channels_in_pages_of_16(cuda, causal, window, new):
    check([1000, 151, 3000], [new, new, new], heads=12, kv_heads=4, dim=128, page=16,
          format="e4m3", causal=causal, window=window)


@pytest.mark.parametrize("format", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_and_read_at_128_channels_in_pages_of_16(cuda, format, dtype):
    before, new, heads, page = [0, 17, 100, 31], [40, 1, 0, 129], 3, 16
    lengths = [o + n for o, n in zip(before, new)]
    width = max(-(-n // page) for n in lengths)
    order = torch.randperm(4 * width, generator=torch.Generator().manual_seed(0)).int()
    table = order.view(4, width).to("cuda")
    cache = QuantizedCache(4 * width, heads, 128, page_size=page, format=format)
    g = torch.Generator(device="cuda").manual_seed(1)
    codes, scales = cache.codes.clone(), cache.scales.clone()
    for counts, ends in ((before, before), (new, lengths)):
        k, v = (torch.randn(sum(counts), heads, 128, generator=g, device="cuda").to(dtype)
                for _ in range(2))
        cache.append(k, v, table, ints(ends), offsets_of(counts), max_tokens=max(counts))
        codes, scales = appended(codes, scales, table, ends, counts, k, v, format)
    cache.check()
    assert cache.codes.dtype == CODE[format] and torch.equal(raw(cache.codes), raw(codes))
    assert torch.equal(cache.scales, scales)
    k, v = cache.read(table, ints([0] * 4), offsets_of(lengths), total=sum(lengths), dtype=dtype)
    at = 0
    for b, n in enumerate(lengths):
        for got, want in zip((k, v), tokens_of(codes, scales, table, b, 0, n)):
            assert torch.equal(got[at:at + n], want.transpose(0, 1).float().to(dtype))
        at += n


@pytest.mark.parametrize("format", ["e4m3", "int8"])
def test_a_page_written_token_by_token_against_its_values(cuda, format):
    """Older codes are rounded again whenever a larger token comes: after token t
    of n that happens 1 / (t + 1) + ... + 1 / n times, on average over t once,
    each with at most the final step's variance. The rms error is therefore at
    most sqrt 2 times that of the same page written at once (1.5 with the
    spread of 128 pages)."""
    pages, page = 128, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(pages, page, 1, 64, generator=g, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[:, None]
    whole, slow = (QuantizedCache(pages, 1, 64, page_size=page, format=format) for _ in range(2))
    flat = x.flatten(0, 1)
    whole.append(flat, flat, table, ints([page] * pages), offsets_of([page] * pages))
    for t in range(page):
        slow.append(x[:, t], x[:, t], table, ints([t + 1] * pages))
    rms = []
    for cache in (whole, slow):
        k, _ = cache.read(table, ints([0] * pages), offsets_of([page] * pages),
                          total=pages * page, dtype=torch.float32)
        cache.check()
        rms.append((k - flat).square().mean().sqrt().item())
    print(f"{format}: {rms[0]:.4f} at once, {rms[1]:.4f} token by token ({rms[1] / rms[0]:.2f})")
    assert rms[0] <= rms[1] <= 1.5 * rms[0]
