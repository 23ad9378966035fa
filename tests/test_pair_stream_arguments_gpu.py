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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 66, 67, 68])
def test_the_addition_keeps_subnormals(d, dtype):
    """Multiples of the smallest subnormal add up, and double where half of them are kept, without rounding."""
    p = P()
    step = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}[dtype]
    u, r = ((torch.randint(-40, 41, (1, 3, 5, d), device=DEV).double() * step).to(dtype) for _ in range(2))
    assert torch.equal(p.dropout_add(u, r), (u.double() + r.double()).to(dtype)) and (u != 0).any()
    drop = p.PairDropout(0.5, seed=3)
    kept = p.dropout_add(torch.ones_like(u), None, drop) != 0
    want = torch.where(kept, u.double() * 2, 0.0)
    assert torch.equal(p.dropout_add(u, None, drop), want.to(dtype))
    assert torch.equal(p.dropout_add(u, r, drop), (want + r.double()).to(dtype))
    w = torch.ones(d, device=DEV)
    assert torch.equal(p.add_rms_norm(u, r, w, dropout=drop)[1], (want + r.double()).to(dtype))
    table, index = u[0, :, 0].contiguous(), torch.tensor([2, -1, 0, 1, 2], device=DEV)
    want = torch.where((index >= 0)[:, None], table.double()[index.clamp(min=0)], 0.0) * 2 + r[0, 0].double()
    assert torch.equal(p.pair_embedding(index, table, scale=2.0, base=r[0, 0]), want.to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 128, 384, 512, 1024, 8192, 66, 130, 131, 132, 1031, 4099])
def test_the_stream_has_the_same_bits_in_every_form(d, dtype):
    """fp32 product, fp32 sum, one rounding to the type: whatever the width and the boundaries (every rank of a grid has to store what one
    GPU would), in the addition and in each norm."""
    p = P()
    drop = p.PairDropout(0.25, seed=3)
    gain = torch.tensor(65536 / 49152, dtype=torch.float32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(d)
    flat = [torch.randn(3 * 7 * d + 1, generator=g, device=DEV).to(dtype) for _ in range(2)]
    w = torch.ones(d, device=DEV)
    for first in (0, 1):
        u, r = (t[first:first + 3 * 7 * d].view(1, 3, 7, d) for t in flat)
        kept = p.dropout_add(torch.ones_like(u), None, drop) != 0
        want = (torch.where(kept, u.float() * gain, 0.0) + r.float()).to(dtype)
        for z in (p.dropout_add(u, r, drop), p.add_rms_norm(u, r, w, dropout=drop)[1], p.add_rms_norm_fp8(u, r, w, group=None, dropout=drop)[2]):
            assert torch.equal(z, want)
