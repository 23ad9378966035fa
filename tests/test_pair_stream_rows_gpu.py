"""Every kernel form over more rows than the device holds at once, so that its loop over rows runs more than one step, with a ragged
end; all rows against the 64-bit oracle.

An SM has 2048 threads, so at most 2048 / lanes of its rows are at hand at once, and 148 SMs have 148 x 2048 / lanes.  2.3 times as many
rows, an odd number, make two or three steps.  (Each lane takes at most 16 channels, so lanes >= D / 16, and rows of up to 64 channels have 8.)

Tolerances as in test_pair_stream_gpu.py; rows above 4096 channels are joined in 10 steps, five in a warp and five over 32 warps:
16 + 10 roundings of 2^-24 in a row's sum, fewer than the 40 that are counted there.  A gain's gradient is summed in fp32 over 32
rows and in 64 bits from there: 32 + 8 roundings, 2^-18 of the absolute values."""
import functools

import pytest
import torch

from oracle.pair_oracle import dropped, embedding, embedding_grad, keep_mask, rms_norm, rms_norm_grad

from .test_pair_stream_gpu import TYPES, near, rand

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
# whole octs; two channels at a time (16-bit types; of fp32 one); one at a time
WIDTHS = (64, 128, 256, 384, 512, 520, 1024, 2048, 4096, 8192) + (66, 130, 500, 1030, 4098) + (67, 131, 187, 253, 401, 1031, 2051, 4099, 8191)


def P():
    from fold_cp_ops_b200.workflows import pair_stream

    return pair_stream


def lanes_of(d, octs):
    """Lanes of a row, from below."""
    if octs:
        return next(n for n, most in ((8, 64), (16, 128), (16, 384), (32, 512), (128, 1024), (256, 2048), (512, 4096), (1024, 8192)) if d <= most)
    return next(n for n, most in ((32, 256), (64, 512), (128, 1024), (256, 2048), (512, 4096), (1024, 8192)) if d <= most)


def shape_of(d):
    rows = int(2.3 * 148 * 2048 / lanes_of(d, d % 8 == 0)) | 1
    j = 61
    return (1, rows // j + 1, j, d)


@functools.lru_cache(maxsize=1)
def mask_of(d):
    return keep_mask(shape_of(d), 0.25, 31, 0, "rows")


def inputs(d, dtype, layout):
    shape = shape_of(d)
    if layout == "block":  # rows that do not follow one another, 16-byte aligned where D is
        u = rand(1, shape[1] + 1, shape[2] + 2, d, dtype=dtype, seed=1)[:, 1:, 2:]
    else:
        u = rand(*shape, dtype=dtype, seed=1)
    return u, rand(*shape, dtype=dtype, seed=2), (1 + rand(d, seed=3, scale=0.1)).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_norm_and_gradients(d, dtype):
    p = P()
    for k, layout in enumerate(("whole", "block")):
        u, r, w = inputs(d, dtype, layout)
        drop, mask_gain = (p.PairDropout(0.25, seed=31, shared="rows"), mask_of(d)) if k else (None, None)
        leaves = [t.detach().requires_grad_() for t in (u, r, w)]
        y, z = p.add_rms_norm(*leaves, dropout=drop)
        du = u.double() if mask_gain is None else dropped(u, *mask_gain)
        near(z.detach(), du + r.double(), du.abs() + r.double().abs(), f"{layout} z", 2.0 ** -22)
        y64 = rms_norm(z.detach(), w, 1e-5)
        near(y.detach(), y64, y64.abs(), f"{layout} y", 2.0 ** -18)
        dy, dz = rand(*u.shape, dtype=dtype, seed=21), rand(*u.shape, dtype=dtype, seed=22)
        got = torch.autograd.grad((y, z), leaves, (dy, dz))
        g, g_abs, dw, dw_abs = rms_norm_grad(z.detach(), w, 1e-5, dy, dz)
        near(got[1], g, g_abs, f"{layout} d_residual")
        if mask_gain is not None:
            g, g_abs = dropped(g, *mask_gain), g_abs * mask_gain[1]
        near(got[0], g, g_abs, f"{layout} d_update")
        near(got[2], dw, dw_abs, f"{layout} d_weight")
        assert torch.equal(p.dropout_add(u, r, drop), z)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_norm_in_e4m3(d, dtype):
    """Bounds as in test_pair_stream_gpu.py's test of the e4m3 form."""
    p = P()
    for k, group in enumerate((None, 32, 64, 128)):
        if group is not None and d % group:
            continue
        u, r, w = inputs(d, dtype, ("whole", "block")[k % 2])
        drop = p.PairDropout(0.25, seed=31, shared="rows") if k < 2 else None
        q, scales, z = p.add_rms_norm_fp8(u, r, w, group=group, dropout=drop)
        assert torch.equal(z, p.dropout_add(u, r, drop))
        n = group or d
        y64 = rms_norm(z, w, 1e-5).unflatten(-1, (d // n, n))
        want = y64.abs().amax(-1) / 448.0
        assert ((scales.double() - want).abs() <= 2.0 ** -17 * want).all()
        unit = y64 / scales.double()[..., None]
        err = (q.float().double().reshape(unit.shape) - unit).abs()
        assert (err <= torch.maximum(2.0 ** -4 * unit.abs(), torch.full_like(unit, 2.0 ** -10)) * (1 + 2.0 ** -15)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [264, 66, 67, 300, 301])
def test_addition_and_embedding(d, dtype):
    """A warp takes 256 channels of a row, or 32 octs: 148 x 64 warps at once, and 2.5 times as many pieces or more."""
    p = P()
    shape = (1, 401, 61, d)
    u, r = rand(*shape, dtype=dtype, seed=1), rand(1, 402, 63, d, dtype=dtype, seed=2)[:, 1:, 1:62]
    mask, gain = keep_mask(shape, 0.25, 31, 0, "columns")
    du = dropped(u, mask, gain)
    drop = p.PairDropout(0.25, seed=31, shared="columns")
    near(p.dropout_add(u, r, drop), du + r.double(), du.abs() + r.double().abs(), "dropout", 2.0 ** -22)
    near(p.dropout_add(u, r), u.double() + r.double(), u.double().abs() + r.double().abs(), "addition", 2.0 ** -22)
    table = rand(50, d, dtype=dtype, seed=3).requires_grad_()
    index = torch.randint(-1, 51, shape[:3], device=DEV)
    out = p.pair_embedding(index, table, scale=0.5, base=u)
    want = embedding(index, table.detach(), u, 0.5)
    near(out.detach(), want, (want - u.double()).abs() + u.double().abs(), "embedding", 2.0 ** -22)
    (got,) = torch.autograd.grad(out, table, r)
    near(got, *embedding_grad(index, 50, r, 0.5), "its gradient", 2.0 ** -13)
