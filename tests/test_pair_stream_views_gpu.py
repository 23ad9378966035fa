"""Views with axes of one entry, whose strides torch leaves as they were."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def P():
    from fold_cp_ops_b200.workflows import pair_stream

    return pair_stream


def views(dtype, d=128):
    g = torch.Generator(device=DEV).manual_seed(5)

    def rand(*shape):
        return torch.randn(shape, generator=g, device=DEV).to(dtype)

    n = 6 * 7 * d
    odd = rand(3, n + 3)[:, :n].unflatten(1, (6, 7, d))
    wide = rand(2, 8, 4, d + 3)[..., :d]  # whole rows of b = 8 x 4 x (d + 3) elements, odd ones inside
    return {"one batch": odd[:1], "one row": odd[:1, :1], "one column": odd[:1, :, :1], "one position of each": wide[:, :1, :1],
            "one position": wide[1:, 3:4, 2:3], "one row of each": rand(2, 9, 7, d)[:, 4:5], "one column of each": rand(3, 5, 7, d)[:, :, 6:]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("name", ["one batch", "one row", "one column", "one position of each", "one position", "one row of each", "one column of each"])
def test_axes_of_one_entry(name, dtype):
    """The same bits as for a copy: the strides of such axes choose nothing.  (Rows that are themselves off 16-byte boundaries -- here
    position 1834 of a tensor, 3668 bytes on -- are added up in another order, by two channels at a time: then the scales agree to
    2^-17 and q to a step of e4m3.)"""
    p, x = P(), views(dtype)[name]
    copy, w = x.clone(memory_format=torch.contiguous_format), torch.linspace(0.5, 1.5, 128, device=DEV)
    whole = x.data_ptr() % 16 == 0 and all(n == 1 or s * x.element_size() % 16 == 0 for n, s in zip(x.shape[:3], x.stride()))
    drop = p.PairDropout(0.25, seed=3)
    for group in (None, 32, 64, 128):
        got, want = p.add_rms_norm_fp8(x, x, w, group=group), p.add_rms_norm_fp8(copy, copy, w, group=group)
        if whole or group is not None:
            assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))
        else:
            a, b = got[0].float(), want[0].float()
            assert torch.equal(got[2], want[2]) and ((got[1] - want[1]).abs() <= 2.0 ** -17 * want[1]).all()
            assert ((a - b).abs() <= torch.maximum(2.0 ** -3 * b.abs(), torch.full_like(b, 2.0 ** -9))).all()
    assert torch.equal(p.dropout_add(x, x, drop), p.dropout_add(copy, copy, drop))
    outs = []
    for t in (x, copy):
        u, v = t.detach().requires_grad_(), w.clone().requires_grad_()
        y, z = p.add_rms_norm(u, t, v, dropout=drop)
        outs.append((y, z, *torch.autograd.grad((y, z), (u, v), (t, t))))
    if whole:
        assert all(torch.equal(a, b) for a, b in zip(*outs))
