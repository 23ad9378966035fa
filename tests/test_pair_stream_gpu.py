"""The pair-stream operators on the GPU against their 64-bit oracle.

Tolerances count roundings.  A result is rounded once to its type, off by at most eps/2 of its value (eps/2 = 2^-8, 2^-11,
2^-24 for bf16, fp16, fp32).  Before that everything is fp32 with unit roundoff 2^-24: a sum of a row has at most 32 terms
per lane and 8 joining steps (40 x 2^-24 of the sum of absolute values), its reciprocal root is off by another 2^-22, and
five products follow, so a norm's value is off by less than 64 x 2^-24 = 2^-18 of it and a gradient by less than 2^-17 of the
sum of the absolute values of its terms."""
import gc

import pytest
import torch

from oracle.pair_oracle import dropped, embedding, embedding_grad, keep_mask, rms_norm, rms_norm_grad

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = (torch.bfloat16, torch.float16, torch.float32)
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}  # half a subnormal step, or flushed


def P():
    from fold_cp_ops_b200.workflows import pair_stream

    return pair_stream


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed + 17 * len(shape) + sum(shape))
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def layouts(shape, dtype, seed, layout):
    B, I, J, D = shape
    if layout == "block":      # a block of a larger tensor
        return rand(B, I + 2, J + 1, D, dtype=dtype, seed=seed)[:, 1:I + 1, 1:]
    if layout == "transposed":  # the incoming update's view
        return rand(B, J, I, D, dtype=dtype, seed=seed).transpose(1, 2)
    if layout == "broadcast":  # one row for all i
        return rand(B, 1, J, D, dtype=dtype, seed=seed).expand(shape)
    if layout == "channels":   # channels are not contiguous
        return rand(B, I, D, J, dtype=dtype, seed=seed).transpose(2, 3)
    if layout == "shifted":    # every row starts two or four bytes off a 16-byte boundary
        return rand(B * I * J * D + 1, dtype=dtype, seed=seed)[1:].view(shape)
    return rand(*shape, dtype=dtype, seed=seed)


def near(got, want, terms, what, fp32=2.0 ** -17):
    """|got - want| <= eps/2 |want| + fp32 * terms, element by element, and no NaN."""
    assert got.dtype in HALF
    err = (got.double() - want).abs()
    bound = HALF[got.dtype] * want.abs() * (1 + fp32) + fp32 * terms + TINY[got.dtype]
    assert bool((err <= bound).all()), f"{what}: {(err - bound).max().item():.3g} beyond the bound, max err {err.max().item():.3g}"


SHAPES = [(1, 1, 1, 1), (1, 1, 1, 512), (1, 5, 7, 8), (2, 3, 5, 64), (1, 9, 11, 128), (1, 4, 6, 256), (1, 3, 7, 384), (1, 3, 5, 520),
          (1, 2, 3, 1024), (1, 1, 5, 2048), (1, 1, 3, 4096), (1, 1, 2, 8192), (2, 3, 4, 131), (1, 3, 2, 1031), (1, 2, 2, 4099),
          (1, 33, 65, 48)]


# ------------------------------------------------------------------------------------------------
# dropout and addition
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_dropout_add(shape, dtype):
    p = P()
    u, r = rand(*shape, dtype=dtype, seed=1), rand(*shape, dtype=dtype, seed=2)
    for k, shared in enumerate((None, "rows", "columns")):
        drop = p.PairDropout(0.25, seed=(1 << 63) + 5, offset=k, shared=shared, origin=(3, 70000, 11))
        mask, gain = keep_mask(shape, 0.25, (1 << 63) + 5, k, shared, (3, 70000, 11))
        du = dropped(u, mask, gain)
        near(p.dropout_add(u, r, drop), du + r.double(), du.abs() + r.double().abs(), f"{shape} {shared}", 2.0 ** -22)
        alone = p.dropout_add(u, None, drop)
        near(alone, du, du.abs(), "without a residual", 2.0 ** -22)
        assert torch.equal(alone != 0, mask.to(DEV) & (u != 0))
    near(p.dropout_add(u, r), u.double() + r.double(), u.double().abs() + r.double().abs(), "no dropout", 2.0 ** -22)


@pytest.mark.parametrize("layout", ["block", "transposed", "broadcast", "channels", "shifted"])
@pytest.mark.parametrize("d", [128, 67])
def test_dropout_add_reads_strided_inputs(layout, d):
    p, shape = P(), (2, 6, 9, d)
    drop = p.PairDropout(0.5, seed=9, shared="rows")
    mask, gain = keep_mask(shape, 0.5, 9, 0, "rows")
    for dtype in TYPES:
        u, r = layouts(shape, dtype, 3, layout), layouts(shape, dtype, 4, "whole" if layout == "shifted" else layout)
        du = dropped(u, mask, gain)
        near(p.dropout_add(u, r, drop), du + r.double(), du.abs() + r.double().abs(), layout, 2.0 ** -22)


def test_every_split_of_the_grid_draws_the_same_mask():
    p = P()
    u = rand(2, 12, 16, 72, dtype=torch.bfloat16, seed=5)
    for shared in (None, "rows", "columns"):
        whole = p.dropout_add(u, None, p.PairDropout(0.3, seed=77, offset=2, shared=shared))
        for i in range(0, 12, 4):
            for j in range(0, 16, 8):
                part = p.dropout_add(u[:, i:i + 4, j:j + 8], None,
                                     p.PairDropout(0.3, seed=77, offset=2, shared=shared, origin=(0, i, j)))
                assert torch.equal(part, whole[:, i:i + 4, j:j + 8])
        assert torch.equal(p.dropout_add(u[1:], None, p.PairDropout(0.3, seed=77, offset=2, shared=shared, origin=(1, 0, 0))), whole[1:])


def test_dropped_infinities_and_nan_become_zero():
    p, shape = P(), (1, 4, 8, 64)
    mask, _ = keep_mask(shape, 0.5, 4)
    u = rand(*shape, seed=6)
    bad = u.masked_fill(~mask.to(DEV), float("nan"))
    bad[0, 0][~mask[0, 0].to(DEV)] = float("inf")
    drop = p.PairDropout(0.5, seed=4)
    assert torch.equal(p.dropout_add(bad, None, drop), p.dropout_add(u, None, drop))
    everything = p.dropout_add(torch.full_like(u, float("nan")), u, p.PairDropout(1.0, seed=4))
    assert torch.equal(everything, u)


def test_in_place_and_refused_overlaps():
    p = P()
    u, r = rand(1, 5, 6, 128, dtype=torch.bfloat16, seed=7), rand(1, 5, 6, 128, dtype=torch.bfloat16, seed=8)
    drop = p.PairDropout(0.25, seed=1)
    want = p.dropout_add(u, r, drop)
    s = r.clone()
    assert p.dropout_add(u, s, drop, out=s) is s and torch.equal(s, want)
    s = u.clone()
    assert torch.equal(p.dropout_add(s, r, drop, out=s), want)
    buf = torch.zeros(2, 5, 6, 128, dtype=torch.bfloat16, device=DEV)
    flat = buf.view(-1)
    for out, x in ((flat[8:8 + u.numel()].view_as(u), flat[:u.numel()].view_as(u)),
                   (u, u.expand_as(u)[:, :, :1].expand_as(u))):
        with pytest.raises(ValueError, match="overlaps"):
            p.dropout_add(x, None, drop, out=out)


def test_out_counts_as_a_change_of_its_tensor():
    p = P()
    u, z = rand(2, 3, 16, seed=9), rand(2, 3, 16, seed=10)
    w = torch.ones(16, device=DEV, requires_grad=True)
    y = (z * w).sum()  # saves z
    with torch.no_grad():
        p.dropout_add(u, z, out=z)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        x = z + 0
        assert torch.equal(p.dropout_add(u, x, out=x), u + z)
    assert torch.equal(p.dropout_add(u, x, out=x), u + (u + z))


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_gradient(dtype):
    p, shape = P(), (2, 5, 6, 72)
    u, r = (rand(*shape, dtype=dtype, seed=s).requires_grad_() for s in (1, 2))
    dz = rand(*shape, dtype=dtype, seed=3)
    mask, gain = keep_mask(shape, 0.25, 3, 1, "columns")
    du, dr = torch.autograd.grad(p.dropout_add(u, r, p.PairDropout(0.25, seed=3, offset=1, shared="columns")), (u, r), dz)
    want = dropped(dz, mask, gain)
    near(du, want, want.abs(), "update", 2.0 ** -22)
    assert torch.equal(dr, dz)
    # the operator is linear in the update: a difference along dz gives the same as the gradient, up to roundings
    ones = torch.ones(1, 1, 1, 72, dtype=dtype, device=DEV).expand(shape)
    (du,) = torch.autograd.grad(p.dropout_add(u, r, p.PairDropout(0.25, seed=3)).sum(), (u,))
    assert torch.equal(du, p.dropout_add(ones, None, p.PairDropout(0.25, seed=3)))


# ------------------------------------------------------------------------------------------------
# the norm
# ------------------------------------------------------------------------------------------------
def check_norm(u, r, w, eps, drop, mask_gain, what, *, grads=True):
    """Forward and gradients against the oracle."""
    p = P()
    u0 = u.double() if mask_gain is None else dropped(u, *mask_gain)
    z64 = u0 if r is None else u0 + r.double()
    terms = u0.abs() if r is None else u0.abs() + r.double().abs()
    leaves = [t.detach().requires_grad_(grads) for t in (u, r, w) if t is not None]
    ur = leaves[:-1] + ([None] if r is None else [])
    y, z = p.add_rms_norm(ur[0], ur[1], leaves[-1], eps=eps, dropout=drop)
    near(z.detach(), z64, terms, f"{what} z", 2.0 ** -22)
    y64 = rms_norm(z.detach(), w, eps)
    near(y.detach(), y64, y64.abs(), f"{what} y", 2.0 ** -18)
    if not grads:
        return
    dy, dz = rand(*u.shape, dtype=u.dtype, seed=21), rand(*u.shape, dtype=u.dtype, seed=22)
    got = torch.autograd.grad((y, z), leaves, (dy, dz))
    g, g_abs, dw, dw_abs = rms_norm_grad(z.detach(), w, eps, dy, dz)
    if mask_gain is None:
        near(got[0], g, g_abs, f"{what} d_update")
    else:
        near(got[0], dropped(g, *mask_gain), g_abs * mask_gain[1], f"{what} d_update")
    if r is not None:
        near(got[1], g, g_abs, f"{what} d_residual")
    near(got[-1], dw, dw_abs, f"{what} d_weight")
    # one output's gradient alone
    for k in (0, 1):
        y, z = p.add_rms_norm(ur[0], ur[1], leaves[-1], eps=eps, dropout=drop)
        got = torch.autograd.grad((y, z)[k], leaves, (dy, dz)[k], allow_unused=True)
        zero = torch.zeros_like(dy)
        g, g_abs, dw, dw_abs = rms_norm_grad(z.detach(), w, eps, zero if k else dy, dz if k else zero)
        want = g if mask_gain is None else dropped(g, *mask_gain)
        near(got[0], want, g_abs * (1 if mask_gain is None else mask_gain[1]), f"{what} d_update of one output")
        if got[-1] is not None:
            near(got[-1], dw, dw_abs, f"{what} d_weight of one output")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_add_rms_norm(shape, dtype):
    u, r = rand(*shape, dtype=dtype, seed=11), rand(*shape, dtype=dtype, seed=12, scale=3.0)
    for wdtype in {dtype, torch.float32}:
        w = (1 + rand(shape[3], seed=13, scale=0.2)).to(wdtype)
        check_norm(u, r, w, 1e-5, None, None, f"{shape} {dtype}")
        check_norm(u, None, w, 1e-5, None, None, f"{shape} {dtype} no residual")
        drop = P().PairDropout(0.2, seed=31, shared="rows")
        check_norm(u, r, w, 1e-5, drop, keep_mask(shape, 0.2, 31, 0, "rows"), f"{shape} {dtype} dropout")
    check_norm(u, None, w, 1e-5, drop, keep_mask(shape, 0.2, 31, 0, "rows"), f"{shape} {dtype} dropout alone")


@pytest.mark.parametrize("layout", ["block", "transposed", "broadcast", "channels", "shifted"])
@pytest.mark.parametrize("d", [256, 67])
def test_norm_reads_strided_inputs(layout, d):
    shape = (2, 6, 9, d)
    for dtype in TYPES:
        u, r = layouts(shape, dtype, 3, layout), layouts(shape, dtype, 4, "whole" if layout == "shifted" else layout)
        w = (1 + rand(d, seed=13, scale=0.2)).to(dtype)
        check_norm(u, r, w, 1e-5, None, None, layout)
        check_norm(u, None, w, 1e-5, None, None, layout)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_many_rows(dtype):
    """More rows than the grid holds at once, several folds of the gain's gradient per CTA, a ragged end."""
    shape = (1, 311, 331, 128)
    u, r, w = rand(*shape, dtype=dtype, seed=1), rand(*shape, dtype=dtype, seed=2), (1 + rand(128, scale=0.1)).to(dtype)
    check_norm(u, r, w, 1e-5, None, None, "many rows")
    first = [t.clone() for t in torch.autograd.grad(P().add_rms_norm(u.requires_grad_(), r, w.requires_grad_())[0].sum(), (u, w))]
    again = torch.autograd.grad(P().add_rms_norm(u, r, w)[0].sum(), (u, w))
    assert all(torch.equal(a, b) for a, b in zip(first, again)), "the same inputs have to give the same bits"


def test_norm_edges():
    p, w = P(), torch.ones(96, device=DEV)
    # rows of zeros, with the smallest eps allowed too: y = 0, and gradients stay finite
    for eps in (1e-5, 1.2e-38):
        z = torch.zeros(1, 2, 3, 96, device=DEV, requires_grad=True)
        y, _ = p.add_rms_norm(z, None, w, eps=eps)
        assert torch.equal(y, torch.zeros_like(y))
        if eps == 1e-5:
            (g,) = torch.autograd.grad(y, z, torch.ones_like(y))
            near(g, torch.full_like(g, 1e-5 ** -0.5).double(), torch.full_like(g, 1e-5 ** -0.5).double(), "zero rows")
    # a NaN or an infinity stays in its row
    z = rand(1, 4, 4, 96, seed=3)
    good, _ = p.add_rms_norm(z, None, w)
    z[0, 1, 2, 5], z[0, 3, 3, 0] = float("nan"), float("inf")
    y, _ = p.add_rms_norm(z, None, w)
    bad = torch.zeros(1, 4, 4, dtype=torch.bool, device=DEV)
    bad[0, 1, 2] = bad[0, 3, 3] = True
    assert torch.equal(y[~bad], good[~bad]) and y[0, 1, 2].isnan().all() and y[0, 3, 3, 0].isnan() and (y[0, 3, 3, 1:] == 0).all()
    # empty tensors
    for shape in ((0, 4, 4, 96), (1, 0, 4, 96), (1, 4, 0, 96)):
        e, wg = torch.zeros(shape, device=DEV, requires_grad=True), w.clone().requires_grad_()
        y, z = p.add_rms_norm(e, e, wg, dropout=p.PairDropout(0.5))
        assert y.shape == z.shape == shape
        g, gw = torch.autograd.grad(y.sum() + z.sum(), (e, wg))
        assert g.shape == shape and torch.equal(gw, torch.zeros_like(w))
        assert p.add_rms_norm_fp8(e.detach(), None, w, group=32)[1].shape == (*shape[:3], 3)
    # fewer dims
    x = rand(7, 96, seed=4)
    assert torch.equal(p.add_rms_norm(x, x, w)[0], p.add_rms_norm(x[None, None], x[None, None], w)[0][0, 0])
    assert torch.equal(p.add_rms_norm(x[0], None, w)[0], p.add_rms_norm(x, None, w)[0][0])


def test_the_streams_rounding_and_the_norm_of_the_stored_stream():
    p = P()
    u, r, w = (rand(2, 3, 4, 128, dtype=torch.bfloat16, seed=s) for s in (1, 2, 3))
    y, z = p.add_rms_norm(u, r, w[0, 0, 0].contiguous())
    assert torch.equal(z, (u.float() + r.float()).bfloat16())
    assert torch.equal(y, p.add_rms_norm(z, None, w[0, 0, 0].contiguous())[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [s for s in SHAPES])
def test_add_rms_norm_fp8(shape, dtype):
    """q is within half an e4m3 step of y / scale (2^-4 of the value, 2^-10 where subnormal), the scales within fp32's."""
    p, d = P(), shape[3]
    u, r, w = rand(*shape, dtype=dtype, seed=1), rand(*shape, dtype=dtype, seed=2, scale=3.0), (1 + rand(d, scale=0.3)).to(dtype)
    if d >= 8:
        w[:8] = 0  # a channel that is always zero
    for group in (None, 32, 64, 128):
        if group is not None and d % group:
            with pytest.raises(ValueError, match="group"):
                p.add_rms_norm_fp8(u, r, w, group=group)
            continue
        for drop in (None, p.PairDropout(0.25, seed=3)):
            q, scales, z = p.add_rms_norm_fp8(u, r, w, group=group, dropout=drop)
            y, z2 = p.add_rms_norm(u, r, w, dropout=drop)
            assert torch.equal(z, z2) and q.dtype is torch.float8_e4m3fn
            n = group or d
            y64 = rms_norm(z, w, 1e-5).reshape(*shape[:3], d // n, n)
            top = y64.abs().amax(-1)
            want = torch.where(top > 0, top / 448.0, torch.ones_like(top))
            assert ((scales.double() - want).abs() <= 2.0 ** -17 * want).all()
            unit = y64 / scales.double()[..., None]
            err = (q.float().double().reshape(unit.shape) - unit).abs()
            assert (err <= torch.maximum(2.0 ** -4 * unit.abs(), torch.full_like(unit, 2.0 ** -10)) * (1 + 2.0 ** -15)).all()


@pytest.mark.parametrize("layout", ["block", "transposed", "broadcast", "channels", "shifted"])
def test_fp8_reads_strided_inputs(layout):
    p, shape, w = P(), (2, 6, 9, 192), (1 + rand(192, seed=5, scale=0.1))
    for dtype in TYPES:
        u, r = layouts(shape, dtype, 3, layout), layouts(shape, dtype, 4, "whole" if layout == "shifted" else layout)
        for group in (None, 64):
            got = p.add_rms_norm_fp8(u, r, w, group=group)
            want = p.add_rms_norm_fp8(u.clone(memory_format=torch.contiguous_format), r.clone(memory_format=torch.contiguous_format), w, group=group)
            # the same values in another order of the row's sum: scales within 2^-17, q within a step of e4m3
            assert torch.equal(got[2], want[2]) and ((got[1] - want[1]).abs() <= 2.0 ** -17 * want[1]).all()
            a, b = got[0].float(), want[0].float()
            assert ((a - b).abs() <= torch.maximum(2.0 ** -3 * b.abs(), torch.full_like(b, 2.0 ** -9))).all()


def test_fp8_of_groups_of_zeros_and_bad_rows():
    p, w = P(), torch.ones(128, device=DEV)
    x = rand(1, 2, 2, 128, seed=3)
    x[0, 0, 0] = 0
    x[0, 0, 1, 32:64] = 0
    x[0, 1, 0, 3] = float("nan")
    q, s, _ = p.add_rms_norm_fp8(x, None, w, group=32)
    assert (s[0, 0, 0] == 1).all() and (q[0, 0, 0].float() == 0).all() and s[0, 0, 1, 1] == 1
    assert q[0, 1, 0].float().isnan().all() and (s[0, 1, 0] == 1).all() and not q[0, 1, 1].float().isnan().any()


# ------------------------------------------------------------------------------------------------
# the embedding
# ------------------------------------------------------------------------------------------------
def indices(kind, n, rows, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + n + rows)
    if kind == "one":
        return torch.full((n,), rows - 1, device=DEV, dtype=dtype)
    if kind == "none":
        return torch.full((n,), -1, device=DEV, dtype=dtype)
    x = torch.rand(n, generator=g, device=DEV)
    x = ((x ** 8 if kind == "skewed" else x) * rows).long().clamp(0, rows - 1)
    if kind == "sorted":
        x = x.sort().values
    if kind == "holes":
        x[::3] = torch.tensor([-1, rows, -(1 << 31), (1 << 31) - 1], device=DEV)[torch.arange((n + 2) // 3, device=DEV) % 4]
    return x.to(dtype)


@pytest.mark.parametrize("dtype,table_dtype", [(a, b) for a in TYPES for b in {a, torch.float32, torch.bfloat16}])
@pytest.mark.parametrize("n,rows,d", [(1, 1, 1), (5, 3, 8), (37, 21, 131), (300, 7, 256), (2047, 66, 128), (2500, 66, 264),
                                      (6000, 3000, 64), (3000, 100000, 32), (4097, 2, 1031), (1, 5000, 8192), (40000, 139, 24)])
def test_embedding_and_its_gradient(n, rows, d, dtype, table_dtype):
    """Sums of d_out are fp32 in steps: at most 128 terms, then at most 64, then the parts of 32 warps or of the shares (in 64 bits):
    fewer than 512 roundings of 2^-24, 2^-15 of the absolute values."""
    p = P()
    for k, kind in enumerate(("uniform", "skewed", "sorted", "holes", "one", "none")):
        index = indices(kind, n, rows, torch.int32 if k % 2 else torch.int64)
        table = rand(rows, d, dtype=table_dtype, seed=1).requires_grad_()
        base = rand(n, d, dtype=dtype, seed=2).requires_grad_()
        scale = (1.0, 11.3, -0.5)[k % 3]
        out = p.pair_embedding(index, table, scale=scale, base=base)
        want = embedding(index, table.detach(), base.detach(), scale)
        near(out.detach(), want, (want - base.detach().double()).abs() + base.detach().double().abs(), kind, 2.0 ** -22)
        d_out = rand(n, d, dtype=dtype, seed=3)
        d_table, d_base = torch.autograd.grad(out, (table, base), d_out)
        want, terms = embedding_grad(index, rows, d_out, scale)
        near(d_table, want, terms, f"{kind} gradient", 2.0 ** -15)
        assert torch.equal(d_base, d_out)
        alone = p.pair_embedding(index, table.detach(), scale=scale, dtype=dtype)
        near(alone, embedding(index, table.detach(), None, scale), (want.abs().max() * 0 + embedding(index, table.detach(), None, scale)).abs(), kind, 2.0 ** -22)


@pytest.mark.parametrize("kind", ["uniform", "skewed", "holes", "one"])
@pytest.mark.parametrize("rows", [66, 2047, 2048, 70000])
def test_embedding_gradient_of_many_tokens(rows, kind):
    """Runs that cross many shares of the sorted tokens, one to three digits, and the same bits twice."""
    p, n, d = P(), 300007, 40
    index, table = indices(kind, n, rows, torch.int64), rand(rows, d, seed=1).requires_grad_()
    d_out = rand(n, d, seed=3)
    got = [torch.autograd.grad(p.pair_embedding(index, table), table, d_out)[0] for _ in range(2)]
    want, terms = embedding_grad(index, rows, d_out, 1.0)
    near(got[0], want, terms, kind, 2.0 ** -15)
    assert torch.equal(got[0], got[1])


@pytest.mark.parametrize("kind", ["uniform", "sorted", "skewed", "holes", "one", "none"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,d", [(1025, 1, 1), (1025, 2, 8), (1400, 21, 131), (5000, 74, 66), (5000, 75, 66), (4800, 73, 200), (1700000, 2, 8),
                                      (90001, 66, 64)])
def test_embedding_gradient_of_small_tables(n, rows, d, dtype, kind):
    """The tables that every warp has to itself, and the sizes next to them.  fp32 sums of at most 1024 terms per warp, joined in 64 bits
    and rounded twice: fewer than 2048 roundings of 2^-24, 2^-13 of the absolute values.  Rows of d_out on odd boundaries as well, and
    values at tokens without an embedding that no row may take."""
    p = P()
    index, table = indices(kind, n, rows, torch.int32), rand(rows, d, seed=1, dtype=dtype).requires_grad_()
    for first in (0, 1):
        d_out = rand(n * d + 1, seed=3, dtype=dtype)[first:n * d + first].view(n, d)
        d_out[(index < 0) | (index >= rows)] = float("nan")
        (got,) = torch.autograd.grad(p.pair_embedding(index, table, scale=-0.5), table, d_out)
        want, terms = embedding_grad(index, rows, d_out.nan_to_num(0.0), -0.5)
        near(got, want, terms, kind, 2.0 ** -13)
        (again,) = torch.autograd.grad(p.pair_embedding(index, table, scale=-0.5), table, d_out)
        assert torch.equal(got, again)


@pytest.mark.parametrize("rows", [21, 66, 300, 70000])
def test_embedding_gradient_captured_and_beside_another(rows):
    """Each form of the gradient: two graphs replayed on new indices, one behind the other and on two streams."""
    p, n, d = P(), 5000, 72
    table, d_out = rand(rows, d, seed=1).requires_grad_(), rand(n, d, seed=2)
    index = [indices("uniform", n, rows, torch.int64, seed=k) for k in range(2)]

    def step(x):
        return torch.autograd.grad(p.pair_embedding(x, table), table, d_out)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(index[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in index], []
    for graph, x in zip(graphs, index):
        with torch.cuda.graph(graph):
            outs.append(step(x))
    for seed in (5, 9):
        for k, x in enumerate(index):
            x.copy_(indices("holes", n, rows, torch.int64, seed=seed + k))
        want = [step(x) for x in index]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        terms = embedding_grad(index[0], rows, d_out, 1.0)
        near(outs[0], *terms, "replayed", 2.0 ** -13)


def test_embedding_shapes_and_strides():
    p = P()
    table = rand(10, 48, seed=1, dtype=torch.bfloat16)
    index = torch.arange(60, device=DEV).reshape(1, 6, 10).transpose(1, 2) % 10
    base = rand(1, 6, 10, 48, dtype=torch.float32, seed=2).transpose(1, 2)
    near(p.pair_embedding(index, table, base=base), embedding(index, table, base, 1.0),
         embedding(index, table, None, 1.0).abs() + base.double().abs(), "views", 2.0 ** -22)
    assert p.pair_embedding(index[:, :0], table).shape == (1, 0, 6, 48)
    assert torch.equal(p.pair_embedding(torch.tensor(3, device=DEV), table), table[3])
    t = table.clone().requires_grad_()
    (g,) = torch.autograd.grad(p.pair_embedding(index[:, :0], t).sum(), t)
    assert torch.equal(g, torch.zeros_like(t))
    wide = table.t().contiguous().t().detach().requires_grad_()  # a table with other strides
    (g,) = torch.autograd.grad(p.pair_embedding(index, wide).sum(), wide)
    want, terms = embedding_grad(index, 10, torch.ones(1, 10, 6, 48, device=DEV), 1.0)
    near(g, want, terms, "strided table", 2.0 ** -15)


def test_offsets_beyond_32_bits():
    """Tensors of more than 2^31 elements: the last rows are what a small call gives."""
    p, d = P(), 512
    n = (1 << 31) // d + 77
    x = torch.empty(1, 1, n, d, dtype=torch.bfloat16, device=DEV)
    x.copy_(rand(1, 1, 1, d, dtype=torch.bfloat16, seed=1).expand_as(x))
    x[0, 0, -50:] = rand(50, d, dtype=torch.bfloat16, seed=2)
    w = (1 + rand(d, seed=3, scale=0.1)).bfloat16().requires_grad_()
    drop = p.PairDropout(0.25, seed=5)
    tail = p.PairDropout(0.25, seed=5, origin=(0, 0, n - 50))
    y, z = p.add_rms_norm(x, None, w.detach(), dropout=drop)
    y2, z2 = p.add_rms_norm(x[:, :, -50:], None, w.detach(), dropout=tail)
    assert torch.equal(y[:, :, -50:], y2) and torch.equal(z[:, :, -50:], z2)
    assert torch.equal(p.dropout_add(x, None, drop)[:, :, -50:], z2)
    del y, z
    g = torch.autograd.grad(p.add_rms_norm(x.requires_grad_(), None, w)[0], x, x.detach())[0][:, :, -50:].clone()
    t = x.detach()[:, :, -50:].clone().requires_grad_()
    assert torch.equal(g, torch.autograd.grad(p.add_rms_norm(t, None, w)[0], t, t.detach())[0])
    x = x.detach()
    index = torch.arange(n, device=DEV) % 7
    table = rand(7, d, dtype=torch.bfloat16, seed=6).requires_grad_()
    out = p.pair_embedding(index, table, base=x[0, 0])
    assert torch.equal(out[-50:], p.pair_embedding(index[-50:], table, base=x[0, 0, -50:]))
    x.zero_()
    x[0, 0, -50:] = 1
    (g,) = torch.autograd.grad(out, table, x[0, 0])
    want = torch.bincount(index[-50:], minlength=7)
    assert torch.equal(g, want[:, None].expand(7, d).to(g.dtype))


# ------------------------------------------------------------------------------------------------
# use: refusals, streams, graphs, the operators together
# ------------------------------------------------------------------------------------------------
def test_refusals():
    p = P()
    x, w = rand(1, 2, 3, 64, dtype=torch.bfloat16), torch.ones(64, device=DEV)
    bad = [
        lambda: p.dropout_add(x, x[:, :1]), lambda: p.dropout_add(x, x.float()), lambda: p.dropout_add(x, x.cpu()),
        lambda: p.dropout_add(x.double()), lambda: p.dropout_add(x[None]), lambda: p.dropout_add(x, out=x.float()),
        lambda: p.dropout_add(x.expand(2, 2, 3, 64), out=rand(2, 2, 64, 3, dtype=torch.bfloat16).transpose(2, 3)),
        lambda: p.dropout_add(x.clone().requires_grad_(), out=x), lambda: p.dropout_add(torch.zeros(1, 1, 1, 0, device=DEV)),
        lambda: p.add_rms_norm(x, None, w[:32]), lambda: p.add_rms_norm(x, None, w.double()),
        lambda: p.add_rms_norm(x, None, w.cpu()), lambda: p.add_rms_norm(x, None, w, eps=0.0),
        lambda: p.add_rms_norm(x, None, w, eps=float("nan")), lambda: p.add_rms_norm(torch.zeros(1, 1, 1, 8200, device=DEV), None, torch.ones(8200, device=DEV)),
        lambda: p.add_rms_norm_fp8(x, None, w, group=48), lambda: p.add_rms_norm_fp8(x, None, w, group=128),
        lambda: p.add_rms_norm_fp8(x, None, w.clone().requires_grad_(), group=64),
        lambda: p.pair_embedding(x, x[0, 0]), lambda: p.pair_embedding(torch.zeros(3, device=DEV, dtype=torch.int16), x[0, 0]),
        lambda: p.pair_embedding(torch.zeros(3, device=DEV, dtype=torch.int64), x[0, 0].double()),
        lambda: p.pair_embedding(torch.zeros(3, device=DEV, dtype=torch.int64), x[0, 0, :0]),
        lambda: p.pair_embedding(torch.zeros(3, device=DEV, dtype=torch.int64), x[0, 0], base=x[0, 0, :2]),
        lambda: p.pair_embedding(torch.zeros(3, device=DEV, dtype=torch.int64), x[0, 0], base=x[0, 0], dtype=torch.float32),
        lambda: p.pair_embedding(torch.zeros(3, device=DEV, dtype=torch.int64), x[0, 0], scale=float("inf")),
        lambda: p.PairDropout(0.5, seed=torch.zeros(3, dtype=torch.int64, device=DEV)),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k} was not refused")
    for call in (lambda: p.dropout_add(x, x, 0.5), lambda: p.add_rms_norm(x, x, w, dropout=0.5)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("needs", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
def test_gradients_of_some_inputs_only(needs):
    p = P()
    ts = [rand(1, 3, 4, 72, seed=k) for k in (1, 2)] + [1 + rand(72, seed=3, scale=0.1)]
    for drop in (None, p.PairDropout(0.25, seed=5)):
        every = [t.clone().requires_grad_() for t in ts]
        g = rand(1, 3, 4, 72, seed=4)
        want = torch.autograd.grad(p.add_rms_norm(*every, dropout=drop)[0], every, g)
        some = [t.clone().requires_grad_(bool(n)) for t, n in zip(ts, needs)]
        got = torch.autograd.grad(p.add_rms_norm(*some, dropout=drop)[0], [t for t in some if t.requires_grad], g)
        assert all(torch.equal(a, b) for a, b in zip(got, [w for w, n in zip(want, needs) if n]))
        if not needs[2]:
            some = some[:2]
            z = p.dropout_add(*some, drop)
            got = torch.autograd.grad(z, [t for t in some if t.requires_grad], g)
            assert torch.equal(got[0], p.dropout_add(g, None, drop) if needs[0] else g)


def test_lazily_negated_inputs():
    p = P()
    x = torch.view_as_complex(rand(1, 3, 4, 64, 2, seed=1)).conj().imag
    assert x.is_neg()
    w = torch.ones(64, device=DEV)
    assert torch.equal(p.dropout_add(x, x), 2 * x.clone()) and torch.equal(p.add_rms_norm(x, x, w)[0], p.add_rms_norm(x.clone(), x.clone(), w)[0])
    assert torch.equal(p.pair_embedding(torch.arange(3, device=DEV), x[0, :, 0]), x[0, :, 0].clone())


def test_more_octs_than_32_bits_count():
    """2^34 elements and some: the quotients of a 64-bit unit number."""
    if torch.cuda.mem_get_info()[0] < 50 << 30:
        pytest.skip("needs 50 GB of device memory")
    p, d = P(), 8192
    n = (1 << 34) // d + 5
    row = rand(1, 1, 1, d, dtype=torch.bfloat16, seed=1).expand(1, 1, n, d)
    drop, tail = p.PairDropout(0.25, seed=5), p.PairDropout(0.25, seed=5, origin=(0, 0, n - 9))
    assert torch.equal(p.dropout_add(row, None, drop)[:, :, -9:], p.dropout_add(row[:, :, -9:], None, tail))
    index, table = torch.arange(n, device=DEV) % 7, rand(7, d, dtype=torch.bfloat16, seed=6)
    assert torch.equal(p.pair_embedding(index, table)[-9:], table[index[-9:]])


def test_a_changed_device_seed_is_an_error_in_the_gradient():
    p = P()
    seed = torch.tensor([5, 1], device=DEV)
    u, w = rand(1, 2, 3, 64).requires_grad_(), torch.ones(64, device=DEV)
    drop = p.PairDropout(0.5, seed=seed)
    assert torch.equal(p.dropout_add(u, None, drop), p.dropout_add(u, None, p.PairDropout(0.5, seed=5, offset=1)))
    outs = [p.dropout_add(u, None, drop), p.add_rms_norm(u, u, w, dropout=drop)[0]]
    seed += 1
    for out in outs:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def _step(p, index, table, update, weight, drop, dy, dz):
    """The operators as they follow one another: bins make the stream, an update is dropped into it, its norm is read."""
    z0 = p.pair_embedding(index, table, scale=0.5)
    y, z = p.add_rms_norm(update, z0, weight, dropout=drop)
    z = p.dropout_add(y, z, drop)
    return torch.autograd.grad((y, z), (table, update, weight), (dy, dz)), z.detach()


def test_the_operators_together_and_captured():
    """A training step of all operators: against autograd in 64 bits, and captured with a device seed and replayed on new
    inputs and a new mask, bit for bit what the eager step gives."""
    p = P()
    B, N, D, V = 1, 48, 128, 66
    index = (torch.arange(N, device=DEV)[:, None] - torch.arange(N, device=DEV)[None]).clamp(-32, 32)[None] + 32
    table, weight = rand(V, D, seed=1).requires_grad_(), (1 + rand(D, seed=2, scale=0.1)).requires_grad_()
    update = rand(B, N, N, D, seed=3).requires_grad_()
    dy, dz = rand(B, N, N, D, seed=4), rand(B, N, N, D, seed=5)
    seed = torch.tensor([11, 0], device=DEV)
    drop = p.PairDropout(0.25, seed=seed, shared="rows")
    grads, z = _step(p, index, table, update, weight, drop, dy, dz)
    t, u, w = (x.detach().double().requires_grad_() for x in (table, update, weight))
    mask, gain = keep_mask((B, N, N, D), 0.25, 11, 0, "rows")
    z64 = 0.5 * t[index] + dropped(u, mask, gain)
    y64 = z64 / torch.sqrt(z64.square().mean(-1, keepdim=True) + 1e-5) * w
    z64 = z64 + dropped(y64, mask, gain)
    want = torch.autograd.grad((y64, z64), (t, u, w), (dy.double(), dz.double()))
    for g, ref in zip(grads, want):  # fp32 throughout: norm-wise, a few hundred roundings
        assert (g.double() - ref).norm() <= 2.0 ** -16 * ref.norm()
    assert (z.double() - z64).norm() <= 2.0 ** -18 * z64.norm()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(p, index, table, update, weight, drop, dy, dz)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two captured graphs of the same step
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(p, index, table, update, weight, drop, dy, dz))
        graphs.append(graph)
    for step in range(3):
        with torch.no_grad():
            update.copy_(rand(B, N, N, D, seed=30 + step))
        seed.copy_(torch.tensor([100 + step, step], device=DEV))
        want, wz = _step(p, index, table, update, weight, drop, dy, dz)
        for graph, (got, gz) in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(gz, wz) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_a_capture_beside_a_living_eager_graph_is_refused():
    """The engine would wait for the eager graph's stream in the middle of the capture; the call is refused before anything
    of it is captured, and the same capture works once the graph is gone."""
    p = P()
    x, w = rand(1, 4, 4, 64, seed=1).requires_grad_(), torch.ones(64, device=DEV, requires_grad=True)
    table, index = rand(9, 64, seed=2).requires_grad_(), torch.arange(16, device=DEV).reshape(1, 4, 4) % 9
    calls = {"norm": lambda: p.add_rms_norm(x, None, w)[0], "add": lambda: p.dropout_add(x, x, p.PairDropout(0.5)),
             "embed": lambda: p.pair_embedding(index, table)}
    for name, call in calls.items():
        want = torch.autograd.grad(call().sum(), table if name == "embed" else x)[0]
        alive = call()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
            with torch.cuda.graph(graph):
                call()
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            (got,) = torch.autograd.grad(call().sum(), table if name == "embed" else x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), name


def test_second_derivatives_are_refused_where_they_are_used():
    p = P()
    x, w = rand(1, 2, 3, 64, seed=1).requires_grad_(), torch.ones(64, device=DEV, requires_grad=True)
    table = rand(5, 64, seed=2).requires_grad_()
    for out, leaf in ((p.add_rms_norm(x, None, w)[0], x), (p.dropout_add(x, None, p.PairDropout(0.5)), x),
                      (p.pair_embedding(torch.arange(5, device=DEV), table), table)):
        (plain,) = torch.autograd.grad(out.sum(), leaf, retain_graph=True)
        (g,) = torch.autograd.grad(out.sum(), leaf, create_graph=True)
        assert torch.equal(g, plain)
        with pytest.raises(RuntimeError, match="differentiable once"):
            g.square().sum().backward()


def test_dtensors_on_one_rank(tmp_path):
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import DTensor, Shard, distribute_tensor

    p, started = P(), not dist.is_initialized()
    if started:
        dist.init_process_group("nccl", init_method=f"file://{tmp_path}/store", rank=0, world_size=1, device_id=torch.device(DEV))
    try:
        mesh = init_device_mesh("cuda", (1,))
        x, w = rand(1, 6, 8, 64, seed=1, dtype=torch.bfloat16), torch.ones(64, device=DEV)
        dx, drop = distribute_tensor(x, mesh, (Shard(1),)), p.PairDropout(0.25, seed=3)
        y, z = p.add_rms_norm(dx, dx, w, dropout=drop)
        want = p.add_rms_norm(x, x, w, dropout=drop)
        assert isinstance(y, DTensor) and torch.equal(y.full_tensor(), want[0]) and torch.equal(z.full_tensor(), want[1])
        s = distribute_tensor(x.clone(), mesh, (Shard(1),))
        assert p.dropout_add(dx, s, drop, out=s) is s and torch.equal(s.full_tensor(), want[1])
    finally:
        if started:
            dist.destroy_process_group()


def test_two_streams_at_once():
    p = P()
    shape = (1, 64, 64, 128)
    index = torch.randint(0, 66, shape[:3], device=DEV)
    table, w = rand(66, 128, seed=1).requires_grad_(), torch.ones(128, device=DEV).requires_grad_()
    ins = [(rand(*shape, seed=k).requires_grad_(), rand(*shape, seed=9 + k)) for k in range(2)]

    def one(u, g):
        y, z = p.add_rms_norm(u, p.pair_embedding(index, table), w, dropout=p.PairDropout(0.2, seed=4))
        return torch.autograd.grad((y, z), (u, table, w), (g, g))

    want = [one(*i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = one(*ins[k])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_training_loop_accumulates_into_leaves():
    """`.backward()` into parameters, twice: gradients add up, and shared gradients are not overwritten."""
    p = P()
    u, r = rand(1, 4, 5, 64, seed=1).requires_grad_(), rand(1, 4, 5, 64, seed=2).requires_grad_()
    w = torch.ones(64, device=DEV, requires_grad=True)
    for _ in range(2):
        y, z = p.add_rms_norm(u, r, w)
        (p.dropout_add(y, z) * 0.5).sum().backward()
    y, z = p.add_rms_norm(u, r, w)
    once = torch.autograd.grad((p.dropout_add(y, z) * 0.5).sum(), (u, r, w))
    for t, g in zip((u, r, w), once):
        near(t.grad, 2 * g.double(), 2 * g.double().abs(), "accumulated")
    u.grad.zero_()
    assert r.grad.abs().sum() > 0, "two leaves must not share one gradient"
    gc.collect()
