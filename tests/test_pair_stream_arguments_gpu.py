"""Arguments at the ends of their ranges."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def P():
    from fold_cp_ops_b200.workflows import pair_stream

    return pair_stream


def test_scales_that_are_infinite_in_float32_are_refused():
    p, table, index = P(), torch.zeros(2, 8, device=DEV), torch.tensor([0, -1], device=DEV)
    for scale in (1e39, -1e39, 3.5e38, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            p.pair_embedding(index, table, scale=scale)
    assert torch.equal(p.pair_embedding(index, table, scale=3.4e38), torch.zeros(2, 8, device=DEV))


@pytest.mark.parametrize("shape", [(0, 1 << 31, 3, 8), (1 << 20, 1 << 20, 0, 8), (1 << 17, 0, 1, 8)])
def test_empty_tensors_with_long_axes(shape):
    """No rows, whatever the other axes say (2^17 batch entries are more than a dropout numbers)."""
    p, x, w = P(), torch.empty(shape, device=DEV).requires_grad_(), torch.ones(8, device=DEV, requires_grad=True)
    drop = p.PairDropout(0.5, seed=1)
    y, z = p.add_rms_norm(x, x, w, dropout=drop)
    assert y.shape == z.shape == p.dropout_add(x, x, drop).shape == shape
    g, gw = torch.autograd.grad((y, z), (x, w), (torch.empty_like(y), torch.empty_like(z)))
    assert g.shape == shape and torch.equal(gw, torch.zeros_like(w))
    q, scales, z = p.add_rms_norm_fp8(x.detach(), None, w.detach(), group=None)
    assert q.shape == shape and scales.shape == (*shape[:3], 1) and z.shape == shape
