"""Which packed rows a cache call takes: rows of no user, rows that do not fit."""

import math

import pytest
import torch

from cache8_case import attend, paged
from cxlsparse_b200 import CxsError
from cxlsparse_b200.quantized import QuantizedCache

pytestmark = pytest.mark.gpu

# Offsets of three users in ten packed rows, max_tokens, the user that does not fit.
MISFITS = [([0, 2, 8, 10], 4, 1), ([0, 2, 4, 14], None, 2), ([-2, 2, 4, 10], None, 0)]
LENGTHS = [20, 31, 17]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def raw(t):
    return t.view(torch.uint8)


def scaled(offsets, most, by):
    lengths = [n * by for n in LENGTHS]
    return [o * by for o in offsets], None if most is None else most * by, lengths


def case(by, format, heads=2, dim=64, page=16):
    return paged([n * by for n in LENGTHS], kv_heads=heads, dim=dim, page_size=page, format=format)


@pytest.mark.parametrize("by", [1, 40])
@pytest.mark.parametrize("format", ["e4m3", "int8"])
@pytest.mark.parametrize("offsets,most,misfit", MISFITS)
def test_append_leaves_a_user_whose_rows_do_not_fit(cuda, offsets, most, misfit, format, by):
    """Its pages stay as they were, with the error bit; the others are written."""
    offsets, most, lengths = scaled(offsets, most, by)
    codes, scales, table = case(by, format)
    k, v = (torch.randn(10 * by, 2, 64, device="cuda") for _ in range(2))
    cache = QuantizedCache(codes=codes.clone(), scales=scales.clone())
    cache.append(k, v, table, ints(lengths), ints(offsets), max_tokens=most)
    with pytest.raises(CxsError, match="lengths or offsets"):
        cache.check()
    alone = QuantizedCache(codes=codes.clone(), scales=scales.clone())
    for b in range(3):
        if b != misfit:
            rows = slice(offsets[b], offsets[b + 1])
            alone.append(k[rows], v[rows], table[b:b + 1], ints(lengths[b:b + 1]),
                         ints([0, offsets[b + 1] - offsets[b]]))
    alone.check()
    assert torch.equal(raw(cache.codes), raw(alone.codes))
    torch.testing.assert_close(cache.scales, alone.scales, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("by", [1, 40])
@pytest.mark.parametrize("offsets,most,misfit", MISFITS)
def test_attend_gives_nothing_to_rows_that_do_not_fit(cuda, offsets, most, misfit, by):
    offsets, most, lengths = scaled(offsets, most, by)
    codes, scales, table = case(by, "int8")
    q = torch.randn(10 * by, 4, 64, device="cuda").half()
    nothing = torch.full((10 * by, 4, 64), math.nan, device="cuda").half()
    del nothing                                    # its memory is what the call finds
    cache = QuantizedCache(codes=codes, scales=scales)
    out, lse = cache.attend(q, table, ints(lengths), ints(offsets), max_tokens=most,
                            return_lse=True)
    with pytest.raises(CxsError, match="lengths or offsets"):
        cache.check()
    for b in range(3):
        low, high = max(offsets[b], 0), min(offsets[b + 1], 10 * by)
        if b == misfit:
            assert (out[low:high] == 0).all() and (lse[low:high] == -math.inf).all()
            continue
        want, want_lse, tol, tol_lse = attend(q[low:high], codes, scales, table[b:b + 1],
                                              lengths[b:b + 1], [high - low], causal=True,
                                              window=0, scale=0.125)
        assert ((out[low:high].double() - want).abs() <= tol).all()
        assert ((lse[low:high].double() - want_lse).abs() <= tol_lse).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offsets,most,misfit", MISFITS)
def test_read_gives_zeros_to_rows_that_do_not_fit(cuda, offsets, most, misfit, dtype):
    codes, scales, table = case(1, "int8")
    cache = QuantizedCache(codes=codes, scales=scales)
    garbage = [torch.full((10, 2, 64), math.nan, dtype=dtype, device="cuda") for _ in range(2)]
    del garbage                                    # its memory is what the call finds
    k, v = cache.read(table, ints([0, 1, 2]), ints(offsets), total=10, max_tokens=most,
                      dtype=dtype)
    with pytest.raises(CxsError, match="lengths or offsets"):
        cache.check()
    for b in range(3):
        rows = slice(max(offsets[b], 0), min(offsets[b + 1], 10))
        if b == misfit:
            assert (k[rows] == 0).all() and (v[rows] == 0).all()
            continue
        n = rows.stop - rows.start
        want = cache.read(table[b:b + 1], ints([b]), ints([0, n]), total=n, dtype=dtype)
        assert torch.equal(k[rows], want[0]) and torch.equal(v[rows], want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offsets,most,total", [
    ([0, 3, 5, 9], None, 400),              # rows past the last user's
    ([7, 9, 9, 12], None, 12),              # rows before the first user's
    ([0, 0, 0, 0], 0, 20),                  # no user has any
])
def test_read_writes_every_row(cuda, offsets, most, total, dtype):
    """Rows that no user has are 0."""
    codes, scales, table = case(1, "int8")
    cache = QuantizedCache(codes=codes, scales=scales)
    garbage = [torch.full((total, 2, 64), math.nan, dtype=dtype, device="cuda") for _ in range(2)]
    del garbage                                    # its memory is what the call finds
    k, v = cache.read(table, ints([0, 1, 2]), ints(offsets), total=total, max_tokens=most,
                      dtype=dtype)
    cache.check()
    want = torch.zeros(2, total, 2, 64, dtype=dtype, device="cuda")
    for b in range(3):
        low, high = offsets[b], offsets[b + 1]
        if high > low:
            want[0, low:high], want[1, low:high] = cache.read(
                table[b:b + 1], ints([b]), ints([0, high - low]), total=high - low, dtype=dtype)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_read_of_no_users_is_zero(cuda):
    cache = QuantizedCache(1, 2, 64)
    garbage = [torch.full((40, 2, 64), math.nan, device="cuda") for _ in range(2)]
    del garbage
    none = torch.zeros(0, 1, dtype=torch.int32, device="cuda")
    k, v = cache.read(none, ints([]), ints([0]), total=40, dtype=torch.float32)
    assert (k == 0).all() and (v == 0).all()


def test_rows_without_room_for_any_are_reported(cuda):
    """max_tokens = 0 for a user that has rows: an error, not silence; no error
    where no user has any (packed rows may be padding)."""
    codes, scales, table = case(1, "int8")
    k = torch.randn(3, 2, 64, device="cuda")
    q = torch.randn(3, 4, 64, device="cuda").half()
    cache = QuantizedCache(codes=codes.clone(), scales=scales.clone())
    one = ints([0, 1, 2, 3])
    cache.append(k, k, table, ints(LENGTHS), one, max_tokens=0)
    with pytest.raises(CxsError, match="lengths or offsets"):
        cache.check()
    out, lse = cache.attend(q, table, ints(LENGTHS), one, max_tokens=0, return_lse=True)
    with pytest.raises(CxsError, match="lengths or offsets"):
        cache.check()
    assert (out == 0).all() and (lse == -math.inf).all()
    got, _ = cache.read(table, ints([0, 0, 0]), one, total=3, max_tokens=0)
    with pytest.raises(CxsError, match="lengths or offsets"):
        cache.check()
    assert (got == 0).all()
    # Without offsets every user has a row: refused before the launch.
    for call in (lambda: cache.append(k, k, table, ints(LENGTHS), max_tokens=0),
                 lambda: cache.attend(q, table, ints(LENGTHS), max_tokens=0),
                 lambda: cache.read(table, ints([0, 0, 0]), None, total=3, max_tokens=0)):
        with pytest.raises(ValueError, match="max_tokens"):
            call()
    cache.append(k, k, table, ints(LENGTHS), ints([0, 0, 0, 0]), max_tokens=0)
    cache.read(table, ints([0, 0, 0]), ints([0, 0, 0, 0]), total=3, max_tokens=0)
    cache.check()
    assert torch.equal(raw(cache.codes), raw(codes))
