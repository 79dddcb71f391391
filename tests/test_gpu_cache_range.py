"""Attention over the 8-bit cache where the weights of the keys lie far apart.

Probabilities are held in fp16. Each case's rows are compared in norm: rounding
to 11 bits is independent from key to key, so the relative error of out in norm
is that of one probability (2^-11 / sqrt 3), together with the rounding of out
itself (2^-11 / sqrt 3 for fp16) and scores from fp32 sums (below 2^-13): 1e-3
for all three, doubled for a row's luck.
"""

import math

import pytest
import torch

from cache8_case import attend, paged
from cxlsparse_b200.quantized import QuantizedCache

pytestmark = pytest.mark.gpu

LIMIT = 2e-3


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def compare(codes, scales, table, length, q, rows, window=0):
    new = len(q)
    out, lse = QuantizedCache(codes=codes, scales=scales).attend(
        q, table, ints([length]), ints([0, new]), max_tokens=new, window=window,
        return_lse=True)
    want, want_lse, _, tol_lse = attend(q, codes, scales, table, [length], [new], causal=True,
                                        window=window, scale=q.shape[2] ** -0.5)
    off = (out.double() - want)[:rows].norm(dim=-1) / want[:rows].norm(dim=-1)
    assert off.max() <= LIMIT, off.max()
    assert ((lse.double() - want_lse).abs() <= tol_lse)[:rows].all()


@pytest.mark.parametrize("format", ["e4m3", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("length,others", [(16384, 1e-2), (16384, 1e-3), (65536, 1e-3)])
def test_attend_beside_a_dominant_key_without_values(cuda, format, dim, new, length, others):
    """A first token that takes nearly all of the softmax and has V = 0: out is
    what the many other keys add up to, each far below the largest weight."""
    page = 64
    codes, scales, table = paged([length], kv_heads=1, dim=dim, page_size=page, format=format,
                                 spread=0.0)
    scales[..., 1] *= 4096.0                       # out well above fp16's subnormals
    bytes_ = codes.view(torch.uint8)
    bytes_[:, :, 0, :, -1] = 0                     # the last channel of K: the sink's own
    first = table[0, 0].item()
    bytes_[first, 0, :, 0] = 0
    bytes_[first, 0, 0, 0, -1] = 0x7E if format == "e4m3" else 127      # the largest code
    top = 448.0 if format == "e4m3" else 127.0
    g = torch.Generator(device="cuda").manual_seed(length + new)
    q = torch.randn(new, 4, dim, generator=g, device="cuda").half()
    q[..., -1] = 0
    _, rest, _, _ = attend(q, codes, scales, table, [length], [new], causal=True, window=0,
                           scale=dim ** -0.5)
    unit = scales[first, 0, 0].double() * top * dim ** -0.5
    q[..., -1] = ((rest + math.log(1 / others)) / unit).half()
    compare(codes, scales, table, length, q, new)


@pytest.mark.parametrize("format", ["e4m3", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [1, 40])
@pytest.mark.parametrize("ratio", [14, 20, 24])
@pytest.mark.parametrize("first", [True, False])
def test_attend_beside_zeros_of_a_page_with_a_large_scale(cuda, format, dim, heads, ratio, first):
    """A page's V scale is 2^ratio times the others', set by a token that the
    rows do not see (the first of all, outside their window, or the last, after
    them); they see only zeros of that page."""
    page, new = 16, 8
    length, window = (1024 + new, 1024) if first else (128, 0)
    codes, scales, table = paged([length], kv_heads=1, dim=dim, page_size=page, format=format,
                                 spread=0.0)
    wide = table[0, 0 if first else length // page - 1].item()
    hidden = 0 if first else page - 1
    codes.view(torch.uint8)[wide, 0, 1, [t for t in range(page) if t != hidden]] = 0
    scales[wide, 0, 1] = scales[table[0, 1], 0, 1] * 2.0 ** ratio
    g = torch.Generator(device="cuda").manual_seed(ratio)
    q = torch.randn(new, heads, dim, generator=g, device="cuda").half()
    compare(codes, scales, table, length, q, new if first else new - 1, window)
