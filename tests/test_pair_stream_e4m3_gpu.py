"""The e4m3 output at its ties: products of 16-bit values over their largest give quotients that lie exactly between two e4m3
values (about one in 2500 elements of random bf16 rows), and those go to the even one.

With p = z w, q = e4m3(y / scale) = e4m3(448 p / max|p|): the row's norm cancels.  For bf16 both factors have 8-bit significands, so p has at
most 16 bits, 448 p = 7 p 64 at most 19, and the quotient of a 19-bit by a 16-bit number is either a tie itself or differs from
it by at least 2^-21 of it (a tie has 5 bits, and 19 + 5 + 16 bits of cross products differ by at least one unit): rounding it
to fp32 first decides nothing.  The oracle's quotient in 64 bits is exact at ties for the same reason."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def P():
    from fold_cp_ops_b200.workflows import pair_stream

    return pair_stream


def quotients(z, w, group):
    """448 p / max|p| per group in 64 bits, and whether it is a tie of two normal e4m3 values."""
    p = (z.double() * w.double()).unflatten(-1, (-1, group))
    top = p.abs().amax(-1, keepdim=True)
    t = torch.where(top > 0, 448.0 * p / top, torch.zeros_like(p))
    m, _ = torch.frexp(t.abs())
    return t.flatten(-2), (((m * 16) % 1 == 0.5) & (t.abs() > 2.0 ** -6)).flatten(-2)


@pytest.mark.parametrize("shape", [(1, 40, 50, 256), (2, 9, 11, 128), (1, 33, 7, 384), (1, 5, 6, 520), (1, 2, 9, 2048), (1, 31, 17, 67),
                                   (1, 17, 31, 130), (1, 3, 5, 1031)])
def test_e4m3_of_bf16_rows_is_that_of_the_exact_quotient(shape):
    p, d = P(), shape[3]
    g = torch.Generator(device=DEV).manual_seed(7 + d)
    u, r = ((torch.randn(shape, generator=g, device=DEV) * s).bfloat16() for s in (0.5, 2.0))
    w = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).bfloat16()
    ties = 0
    for group in (None, 32, 64, 128):
        if group is not None and d % group:
            continue
        q, scales, z = p.add_rms_norm_fp8(u, r, w, group=group)
        t, tie = quotients(z, w, group or d)
        ties += int(tie.sum())
        want = t.float().to(torch.float8_e4m3fn)
        assert torch.equal(q.float(), want.float()), f"group {group}: {(q.float() != want.float()).sum().item()} of {q.numel()} differ"
    assert ties > 0 or u.numel() < 100000


@pytest.mark.parametrize("d", [64, 96, 128, 256, 384, 1024, 4096, 67, 130])
def test_neighbours_of_rows_without_a_norm(d):
    """Rows of zeros, of tiny values and with a NaN or an infinity change nothing in the rows beside them."""
    p = P()
    g = torch.Generator(device=DEV).manual_seed(d)
    z = torch.randn((1, 12, 97, d), generator=g, device=DEV).bfloat16()
    w = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).bfloat16()
    kind = torch.randint(0, 12, z.shape[:3], generator=g, device=DEV)
    z[kind == 0] = 0
    z[kind == 1] *= 2.0 ** -100
    z[..., 5][kind == 2] = float("nan")
    z[..., 7][kind == 3] = float("inf")
    for group in (None, 32, 64, 128):
        if group is not None and d % group:
            continue
        q, scales, _ = p.add_rms_norm_fp8(z, None, w, group=group)
        t, _ = quotients(z, w, group or d)
        plain = kind >= 4
        assert torch.equal(q[plain].float(), t.float().to(torch.float8_e4m3fn).float()[plain]), group
        assert (q[kind == 0].float() == 0).all() and (scales[kind == 0] == 1).all() and q[kind == 2].float().isnan().all() and (scales[kind == 2] == 1).all()
        bad = q[kind == 3].float()
        assert bad[:, 7].isnan().all() and (bad[:, :7] == 0).all() and (bad[:, 8:] == 0).all()
        # tiny rows: half a step of e4m3 and 2^-21 of the quotient
        tiny, got = t[kind == 1], q[kind == 1].float().double()
        assert ((got - tiny).abs() <= torch.maximum(2.0 ** -4 * tiny.abs(), torch.full_like(tiny, 2.0 ** -10)) * (1 + 2.0 ** -16)).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("size", [1e-24, 1e-12, 1.0, 1e12])
def test_e4m3_of_gains_of_every_size(size, dtype):
    """Gains far from one: the scales follow, down to the smallest normal number, and q stays what it is.  Half a step of e4m3 (2^-4 of the
    value, 2^-10 where it is subnormal) and a few roundings of 2^-24."""
    p, d = P(), 96
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn((1, 4, 9, d), generator=g, device=DEV).to(dtype)
    w = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)) * size
    for extra in (1.0, 1e-12):  # 1e-36: the scale's floor
        wx = w * extra
        q, scales, z = p.add_rms_norm_fp8(x, None, wx, group=32)
        z64 = z.double()
        y = z64 / torch.sqrt(z64.square().mean(-1, keepdim=True) + 1e-5) * wx.double()
        y = y.unflatten(-1, (-1, 32))
        want = (y.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
        assert ((scales.double() - want).abs() <= 2.0 ** -20 * want).all()
        t = y / scales.double()[..., None]
        err = (q.float().double().reshape(t.shape) - t).abs()
        # values below 2^-126 are flushed: 2^-126 over a scale of at least 2^-126 is 1
        flushed = 2.0 ** -126 / scales.double()[..., None]
        assert (err <= torch.maximum(2.0 ** -4 * t.abs(), torch.full_like(t, 2.0 ** -10)) * (1 + 2.0 ** -18) + flushed).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 384, 512, 1024, 8192, 67, 130, 1031])
def test_e4m3_of_whole_numbers(d, dtype):
    """z and w of few bits, in every type: products below 2^10, so that quotients are ties or at least 2^-15 away from one (a tie has
    five bits), and one in some 30 is a tie."""
    p = P()
    g = torch.Generator(device=DEV).manual_seed(d)
    z = (torch.randint(-40, 41, (1, 5, 41, d), generator=g, device=DEV) / 8).to(dtype)
    w = (torch.randint(1, 21, (d,), generator=g, device=DEV) / 16).to(dtype)
    for group in (None, 32, 64, 128):
        if group is not None and d % group:
            continue
        q, _, _ = p.add_rms_norm_fp8(z, None, w, group=group)
        t, tie = quotients(z, w, group or d)
        assert tie.sum() > q.numel() / 1000
        assert torch.equal(q.float(), t.float().to(torch.float8_e4m3fn).float()), group
