"""Which packed rows a cache call takes: rows of no user."""

import math

import pytest
import torch

from cache8_case import paged
from cxlsparse_b200.quantized import QuantizedCache

pytestmark = pytest.mark.gpu

LENGTHS = [20, 31, 17]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def case(by, format, heads=2, dim=64, page=16):
    return paged([n * by for n in LENGTHS], kv_heads=heads, dim=dim, page_size=page, format=format)


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
