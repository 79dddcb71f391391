"""The 8-bit cache has no gradient: tensors that need one are refused."""

import pytest
import torch

from cxlsparse_b200.quantized import QuantizedCache


def test_tensors_that_need_a_gradient_are_refused():
    cache = QuantizedCache(4, 2, 64, device="cpu")
    table = torch.zeros(2, 3, dtype=torch.int32)
    lengths = torch.ones(2, dtype=torch.int32)
    k = torch.zeros(2, 2, 64)
    need = torch.zeros(2, 2, 64, requires_grad=True)
    for args in ((need, k), (k, need)):
        with pytest.raises(ValueError, match="gradient"):
            cache.append(*args, table, lengths)
    q = torch.zeros(2, 4, 64, dtype=torch.float16, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        cache.attend(q, table, lengths)


@pytest.mark.gpu
def test_they_are_taken_where_none_is_asked_for(cuda):
    cache = QuantizedCache(4, 2, 64)
    table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    lengths = torch.ones(2, dtype=torch.int32, device="cuda")
    k = torch.randn(2, 2, 64, device="cuda", requires_grad=True)
    q = torch.randn(2, 4, 64, device="cuda").half().requires_grad_()
    with torch.no_grad():
        cache.append(k, k, table, lengths)
        out = cache.attend(q, table, lengths)
    assert not out.requires_grad
    cache.append(k.detach(), k.detach(), table, lengths)
    assert torch.equal(cache.attend(q.detach(), table, lengths), out)
    cache.check()
