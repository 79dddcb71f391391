"""Positions and row counts at the ends of what a cache call takes."""

import pytest
import torch

from cxlsparse_b200.quantized import QuantizedCache

pytestmark = pytest.mark.gpu


def test_append_at_the_last_position_of_more_packed_rows_than_positions(cuda):
    """2^31 - 1 packed rows (all one row, stride 0), of which a user has one, at
    position 2^30 - 1: the pages that a launch of that size would reach lie past
    2^31 positions."""
    page, width = 16, 2 ** 26
    cache = QuantizedCache(2, 1, 64, page_size=page, format="int8")
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    k = torch.linspace(-1, 1, 64, device="cuda").view(1, 1, 64)
    rows = k.expand(2 ** 31 - 1, 1, 64)
    lengths = torch.tensor([2 ** 30], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    cache.append(rows, rows, table, lengths, offsets)
    cache.check()
    starts = lengths - 1
    got, _ = cache.read(table, starts, offsets, total=1, dtype=torch.float32)
    cache.check()
    assert ((got - k).abs() <= 0.51 / 127).all()
    assert (cache.codes[0] == 0).all() and (cache.codes[1, :, :, :-1] == 0).all()
