"""Calls that the pair-stream operators must not answer, refused before they look for a device."""
import pytest
import torch

from fold_cp_ops_b200.workflows import pair_stream as P

X, W = torch.zeros(2, 3, 4, 32), torch.ones(32)
INDEX = torch.zeros(3, dtype=torch.int64)
#: every call with one of its tensors replaced
CALLS = {
    "dropout_add update": lambda t: P.dropout_add(t(X), X),
    "dropout_add residual": lambda t: P.dropout_add(X, t(X), P.PairDropout(0.5)),
    "dropout_add out": lambda t: P.dropout_add(X, X, out=t(X)),
    "add_rms_norm update": lambda t: P.add_rms_norm(t(X), None, W),
    "add_rms_norm residual": lambda t: P.add_rms_norm(X, t(X), W),
    "add_rms_norm weight": lambda t: P.add_rms_norm(X, X, t(W)),
    "add_rms_norm_fp8 update": lambda t: P.add_rms_norm_fp8(t(X), None, W, group=32),
    "add_rms_norm_fp8 residual": lambda t: P.add_rms_norm_fp8(X, t(X), W, group=32),
    "add_rms_norm_fp8 weight": lambda t: P.add_rms_norm_fp8(X, X, t(W), group=32),
    "pair_embedding table": lambda t: P.pair_embedding(INDEX, t(W[None])),
    "pair_embedding base": lambda t: P.pair_embedding(INDEX, W[None], base=t(X[0, :, 0])),
}


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("call", CALLS)
def test_tangents_are_refused(call, requires_grad):
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            CALLS[call](lambda t: forward_ad.make_dual(t.clone().requires_grad_(requires_grad), torch.ones_like(t)))
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            CALLS[call](lambda t: forward_ad.make_dual(t.clone(), torch.ones_like(t)))


@pytest.mark.parametrize("call", ["dropout_add update", "add_rms_norm update", "add_rms_norm_fp8 update", "pair_embedding table"])
def test_tracers_are_refused(call):
    from torch.fx.experimental.proxy_tensor import make_fx

    x = W[None] if "table" in call else X
    with pytest.raises(ValueError, match="cannot be traced"):
        torch.jit.trace(lambda a: CALLS[call](lambda t: a), x)
    with pytest.raises(ValueError, match="cannot be traced"):
        make_fx(lambda a: CALLS[call](lambda t: a))(x)


class Wrapper(torch.Tensor):
    """A subclass that holds another tensor and has no memory itself."""

    @staticmethod
    def __new__(cls, elem):
        out = torch.Tensor._make_wrapper_subclass(cls, elem.shape, dtype=elem.dtype, device=elem.device)
        out.elem = elem
        return out

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        args = [a.elem if isinstance(a, cls) else a for a in args]
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("call", CALLS)
def test_tensors_without_memory_are_refused(call):
    """The library takes a null pointer for an absent tensor: a wrapped residual would be left out without a word."""
    with pytest.raises(ValueError, match="memory of their own"):
        CALLS[call](Wrapper)


def test_an_index_without_memory_is_refused():
    with pytest.raises(ValueError, match="memory of their own"):
        P.pair_embedding(Wrapper(INDEX), W[None])


@pytest.mark.parametrize("kw", [dict(seed=3.0), dict(seed="3"), dict(seed=None), dict(offset=1.5), dict(origin=(0, 0.0, 0)), dict(origin=(0, 0, None)),
                                dict(origin=(0, 0, 1 << 31))])
def test_dropouts_that_are_no_integers_are_refused_where_they_are_made(kw):
    with pytest.raises(ValueError, match="integer"):
        P.PairDropout(0.5, **kw)


def test_integers_of_other_kinds_are_taken():
    import numpy as np

    plain = P._record(P.PairDropout(0.5, seed=7, offset=2, origin=(1, 2, 3)), None)
    other = P.PairDropout(0.5, seed=np.uint64(7), offset=np.int32(2), origin=tuple(torch.tensor([1, 2, 3])))
    assert P._record(other, None) == plain


def test_a_block_behind_the_last_coordinate_is_refused(monkeypatch):
    class Wrap:
        like = None

    monkeypatch.setattr(P, "pair_block_origin", lambda x: (0, 1 << 30, 0))
    assert P._record(P.PairDropout(0.5, origin=(0, (1 << 30) - 1, 0)), Wrap())
    with pytest.raises(ValueError, match="behind"):
        P._record(P.PairDropout(0.5, origin=(0, 1 << 30, 0)), Wrap())
