"""Inputs whose derivative or whose trace would be lost without a word."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_tangents_and_tracers_on_the_device():
    from torch.autograd import forward_ad

    from fold_cp_ops_b200.workflows import pair_stream as p

    x, w = torch.randn(1, 2, 3, 64, device="cuda:0"), torch.ones(64, device="cuda:0")
    calls = [lambda t: p.dropout_add(t, x), lambda t: p.add_rms_norm(x, t, w), lambda t: p.add_rms_norm_fp8(t, x, w, group=64),
             lambda t: p.pair_embedding(torch.arange(3, device="cuda:0"), t[0, 0])]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls:
            with pytest.raises(ValueError, match="forward-mode"):
                call(dual)
            call(forward_ad.unpack_dual(dual).primal)
    for call in calls:
        with pytest.raises(ValueError, match="cannot be traced"):
            torch.jit.trace(call, x)
        call(x)
