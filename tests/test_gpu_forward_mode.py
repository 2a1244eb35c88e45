"""Forward-mode derivatives: no operator computes them, so an input that carries a tangent is refused, whether or not anything requires a
gradient.  Without a check the result would come back without its tangent, which reads as a derivative of zero."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import sphconv_b200 as sphconv
from sphconv_b200.attention import cross_attention
from sphconv_b200.norm import residual_norm, row_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def refused(call, *tensors):
    """call(*tensors) with a tangent on one tensor after the other; it runs without."""
    call(*tensors)
    for grad in (False, True):
        for i in range(len(tensors)):
            with forward_ad.dual_level():
                given = [t.detach().requires_grad_(grad and j != i) for j, t in enumerate(tensors)]
                given[i] = forward_ad.make_dual(given[i], torch.ones_like(given[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*given)
    call(*tensors)


def test_cross_attention():
    ends = [torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (3, 9)]
    q, k, v = (torch.randn(n, 2, 16, device=DEV) for n in (3, 9, 9))
    refused(lambda q, k, v: cross_attention(q, k, v, *ends), q, k, v)


def test_norms():
    rows = [torch.randn(6, 8, device=DEV) for _ in range(3)]
    vectors = [torch.ones(8, device=DEV) for _ in range(5)]
    refused(row_norm, rows[0], *vectors[:2])
    refused(lambda block, residual, gate, weight, bias, scale, next_weight, next_bias:
            residual_norm(block, residual, weight, bias, gate=gate, scale=scale, next_weight=next_weight, next_bias=next_bias),
            *rows, *vectors)


@pytest.mark.parametrize("inference", [False, True])
def test_convolutions(inference):
    idx = torch.tensor([[0, i % 4, i % 5, i % 8] for i in range(20)], dtype=torch.int32, device=DEV)
    x = sphconv.SparseConvTensor(torch.randn(20, 8, device=DEV), [4, 5, 8], 1, indices=idx)
    layer = sphconv.SubMConv3d(8, 16, 3, indice_key="a").to(DEV)

    def run(feature):
        y = sphconv.SparseConvTensor(feature, [4, 5, 8], 1, z_idx=x.z_idx, z_ptr=x.z_ptr)
        with torch.set_grad_enabled(not inference):
            return layer(y)

    run(x.feature)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode|jvp"):
            run(forward_ad.make_dual(x.feature, torch.ones_like(x.feature)))
    run(x.feature)
