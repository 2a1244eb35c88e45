"""What the head's modules check before anything runs on a GPU."""
import pytest
import torch

import sphconv_b200 as sphconv
from sphconv_b200.attention import cross_attention
from sphconv_b200.norm import residual_norm, row_norm


def test_parameters():
    net = sphconv.QueryDecoder(32, 48, heads=4, layers=2, queries=5, key_heads=2, center=True, initial_scale=0.25)
    assert net.queries.shape == (5, 32) and len(net.layers) == 2
    attention = net.layers[0].attention
    assert attention.to_q.weight.shape == (32, 32) and attention.to_kv.weight.shape == (2 * 2 * 8, 48)
    assert net.layers[1].after_mlp.weight is None and bool((net.layers[1].after_mlp.scale == 0.25).all())
    assert set(sphconv.RowNorm(8).state_dict()) == {"weight"}
    assert set(sphconv.RowNorm(8, center=True).state_dict()) == {"weight", "bias"}
    assert set(sphconv.ResidualNorm(8).state_dict()) == {"weight", "next_weight"}


@pytest.mark.parametrize("kw", [dict(heads=4, key_heads=3), dict(heads=0, key_heads=1), dict(heads=4, key_heads=0), dict(heads=5)])
def test_heads_that_do_not_divide(kw):
    with pytest.raises(ValueError, match="multiple"):
        sphconv.CrossAttention(32, 48, **kw)


def test_a_decoder_without_queries_asks_for_them():
    net = sphconv.QueryDecoder(32, 48, heads=4, layers=1)
    assert net.queries is None
    with pytest.raises(ValueError, match="queries"):
        net(None)
    with pytest.raises(ValueError, match="q_ptr"):
        net(None, torch.zeros(3, 32))


def test_there_is_no_cpu_path():
    rows, p = torch.randn(4, 2, 8), torch.tensor([0, 4], dtype=torch.int32)
    for call in (lambda: cross_attention(rows, rows, rows, p, p), lambda: row_norm(rows, torch.ones(8)),
                 lambda: residual_norm(rows, rows, torch.ones(8)), lambda: sphconv.RowNorm(8)(rows)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
