"""``check()`` of the dense 8-bit cache beside other streams."""

import pytest
import torch

from cxlsparse_b200 import CxsError
from cxlsparse_b200.quantized import QuantizedCache

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_check_waits_for_calls_on_other_streams(cuda):
    cache = QuantizedCache(2, 1, 64, page_size=16)
    k = torch.zeros(1, 1, 64, device="cuda")
    bad, length = ints([[7]]), ints([1])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(50_000_000)          # cycles: the call below is still to come
            cache.append(k, k, bad, length)
        with pytest.raises(CxsError, match="page id"):
            cache.check()
        cache.check()
