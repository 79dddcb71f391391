"""NaN values of tokens that a row does not see."""

import pytest
import torch

from cache8_case import attend, offsets_of, paged
from cxlsparse_b200.quantized import QuantizedCache

pytestmark = pytest.mark.gpu

NAN = 0x7F                                         # and 0xFF


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def run(lengths, new, nans, *, heads, kv_heads, dim, page, causal, window, dtype=torch.float16):
    """``nans``: (user, token, KV head, channel) whose V is NaN. Every row that
    sees such a token is NaN in that channel, and everything else is what it is
    with a 0 in its place."""
    codes, scales, table = paged(lengths, kv_heads=kv_heads, dim=dim, page_size=page,
                                 format="e4m3")
    clean = codes.view(torch.uint8).clone()
    dirty = clean.clone()
    group = heads // kv_heads
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randn(sum(new), heads, dim, generator=g, device="cuda").to(dtype)
    expect = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    at = [0] + torch.tensor(new).cumsum(0).tolist()
    for n, (b, token, h, d) in enumerate(nans):
        clean[table[b, token // page], h, 1, token % page, d] = 0
        dirty[table[b, token // page], h, 1, token % page, d] = NAN | (n % 2) << 7
        position = torch.arange(lengths[b] - new[b], lengths[b], device="cuda")
        sees = position >= token if causal else torch.ones_like(position, dtype=torch.bool)
        if window:
            sees = sees & (position - window < token)
        expect[at[b]:at[b + 1], h * group:(h + 1) * group, d] |= sees[:, None]
    args = (table, ints(lengths), offsets_of(new))
    kw = dict(max_tokens=max(new), causal=causal, window=window, return_lse=True)
    out, lse = QuantizedCache(codes=dirty.view(codes.dtype), scales=scales).attend(q, *args, **kw)
    codes = clean.view(codes.dtype)
    plain, plain_lse = QuantizedCache(codes=codes, scales=scales).attend(q, *args, **kw)
    want, _, tol, _ = attend(q, codes, scales, table, lengths, new, causal=causal, window=window,
                             scale=dim ** -0.5)
    assert torch.equal(out.isnan(), expect)
    assert torch.equal(out[~expect], plain[~expect]) and torch.equal(lse, plain_lse)
    assert ((out.double() - want).abs() <= tol)[~expect].all()


@pytest.mark.parametrize("dim,page", [(64, 64), (64, 16), (128, 32), (128, 64)])
@pytest.mark.parametrize("new", [1, 3, 70, 300])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 30), (False, 100), (False, 0)])
def test_attend_nan_values_reach_only_rows_that_see_them(cuda, dim, page, new, causal, window):
    last = 1000
    nans = [(0, last - 1, 0, 5), (0, last - 2, 1, dim - 1), (0, last - new, 0, 33),
            (0, last - 40, 1, 0), (0, last - 31, 0, 17), (0, last - 129, 1, 40),
            (0, max(0, last - new - 20), 0, 63), (1, 77, 1, 12), (1, 0, 0, 1)]
    run([last, 400], [new, min(new, 350)], nans, heads=8, kv_heads=2, dim=dim, page=page,
        causal=causal, window=window)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,new", [(1, 2), (4, 4), (16, 2), (1, 200), (16, 100)])
def test_attend_nan_values_in_items_split_over_ctas(cuda, dim, heads, new):
    """Long histories: an item's parts are joined; the tile that hides keys is in
    one of them."""
    length, window = 40000, 20000
    nans = [(0, length - 1, 0, 3), (0, length - new // 2, 0, dim - 2),
            (0, length - window - new // 2, 0, 9), (0, length - window // 2, 0, 31),
            (0, 5, 0, 50)]
    run([length], [new], nans, heads=heads, kv_heads=1, dim=dim, page=64, causal=True,
        window=window)


@pytest.mark.parametrize("new", [2, 100])
def test_attend_values_that_are_all_nan(cuda, new):
    """The last tokens' V all NaN, many users: rows before them are clean."""
    lengths = [150 + 7 * i for i in range(12)]
    nans = [(b, n - 1 - t, h, d) for b, n in enumerate(lengths) for t in range(2)
            for h in range(2) for d in range(64)]
    run(lengths, [new] * 12, nans, heads=6, kv_heads=2, dim=64, page=16, causal=True, window=0,
        dtype=torch.bfloat16)
