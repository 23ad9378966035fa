"""What the C header promises beyond the Python functions: outputs in the inputs' own memory, and the smallest eps."""
import ctypes as C

import pytest
import torch

from .test_pair_stream_cpu import Dropout, EmbedDesc, NormDesc, Tensor4
from .test_pair_stream_gpu import near, rand

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
KIND = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def P():
    from fold_cp_ops_b200.workflows import pair_stream

    return pair_stream


def call(name, *args):
    from fold_cp_ops_b200 import _lib

    args = [C.byref(a) if isinstance(a, C.Structure) else C.c_void_p(a.data_ptr()) if isinstance(a, torch.Tensor) else C.c_void_p(a) for a in args]
    _lib.check(getattr(_lib.load(), name)(*args, C.c_void_p(torch.cuda.current_stream().cuda_stream)), name)


def tensor4(t):
    return Tensor4(t.data_ptr(), *t.stride()[:3])


@pytest.mark.parametrize("dtype", KIND)
@pytest.mark.parametrize("shape", [(1, 3, 5, 128), (1, 311, 331, 128), (2, 100, 61, 67), (1, 30, 40, 1031), (1, 20, 50, 2048), (2, 30, 70, 384)])
def test_the_stream_in_the_inputs_own_memory(shape, dtype):
    """Norm form and addition: over the residual and over the update, with and without a dropout, in the type and in e4m3."""
    p, (b, i, j, d) = P(), shape
    u, r, w = rand(*shape, dtype=dtype, seed=1), rand(*shape, dtype=dtype, seed=2), 1 + rand(d, seed=3, scale=0.1)
    for keep, drop in ((65536, None), (49152, p.PairDropout(0.25, seed=7, offset=3, shared="rows"))):
        y, z = p.add_rms_norm(u, r, w, dropout=drop)
        q, scales, _ = p.add_rms_norm_fp8(u, r, w, group=None, dropout=drop)
        for own in ("update", "residual"):
            for form in ("add", "norm", "e4m3"):
                desc = NormDesc(b, i, j, d, KIND[dtype], 2, d if form == "e4m3" else 0, 1e-5, Dropout(7, 3, keep, None, 1, 0, 0, 0))
                uu, rr = u.clone(), r.clone()
                to = uu if own == "update" else rr
                yy = torch.empty_like(q if form == "e4m3" else y)
                ss = torch.empty_like(scales)
                norm = form != "add"
                call("pair_sm100_add_norm", desc, tensor4(uu), tensor4(rr), w if norm else None, to, yy if norm else None, ss if form == "e4m3" else None)
                assert torch.equal(to, z), (own, form)
                assert form != "norm" or torch.equal(yy, y)
                assert form != "e4m3" or (torch.equal(yy.float(), q.float()) and torch.equal(ss, scales))


@pytest.mark.parametrize("dtype", KIND)
@pytest.mark.parametrize("n,d", [(5, 8), (90001, 64), (30011, 67)])
def test_the_embedding_over_its_base(n, d, dtype):
    p = P()
    index, table, base = torch.randint(-1, 12, (n,), device=DEV), rand(11, d, dtype=dtype, seed=1), rand(n, d, dtype=dtype, seed=2)
    want = p.pair_embedding(index, table, scale=0.5, base=base)
    call("pair_sm100_embed", EmbedDesc(n, d, 11, 64, KIND[dtype], KIND[dtype], 0.5), index, table, base, base)
    assert torch.equal(base, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [96, 67, 1024])
@pytest.mark.parametrize("eps", [1e-5, 1.2e-38])
def test_gradients_of_rows_of_zeros(eps, d, dtype):
    """g = w dy / sqrt(eps): where sqrt(eps)^-3 overflows too, and the gain's gradient is 0."""
    p = P()
    z, w = torch.zeros(1, 3, 4, d, device=DEV, dtype=dtype).requires_grad_(), (1 + rand(d, seed=1, scale=0.1)).requires_grad_()
    dy = rand(1, 3, 4, d, dtype=dtype, seed=2)
    y, _ = p.add_rms_norm(z, None, w, eps=eps)
    g, gw = torch.autograd.grad(y, (z, w), dy)
    eps32 = torch.tensor(eps, dtype=torch.float32).double().item()
    want = w.detach().double() * dy.double() * eps32 ** -0.5
    near(g, want, want.abs(), "zero rows")
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(gw, torch.zeros_like(w))
