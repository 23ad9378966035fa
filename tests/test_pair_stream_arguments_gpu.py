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
