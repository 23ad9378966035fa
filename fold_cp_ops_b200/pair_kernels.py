"""Per-kernel Python entry points of the pair-stream operators, over the C ABI of ``include/pair_stream_sm100.h``.

As in :mod:`fold_cp_ops_b200.kernels`, each function checks types and layouts, passes device pointers and the
current CUDA stream to the library and writes into tensors that the caller provides (the ``*_workspace`` functions say
how many bytes of scratch to provide).  :mod:`fold_cp_ops_b200.workflows.pair_stream` allocates and differentiates.

Activations are ``(B, N_i, N_j, D)`` tensors of any strides whose channels are contiguous; outputs are contiguous.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib

DTYPES = {torch.bfloat16: _lib.PAIR_BF16, torch.float16: _lib.PAIR_FP16, torch.float32: _lib.PAIR_FP32}
_NULL = _lib.PairTensor()


def _kind(t: torch.Tensor, name: str) -> int:
    kind = DTYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"{name} must be bfloat16, float16 or float32; got {t.dtype}")
    return kind


def _cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor; the pair-stream kernels have no CPU path")


def _view(t: Optional[torch.Tensor], like: torch.Tensor, name: str) -> _lib.PairTensor:
    """The pointer and strides of a tensor shaped and typed as ``like``."""
    if t is None:
        return _NULL
    if t.shape != like.shape or t.dtype is not like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {tuple(like.shape)} {like.dtype} on {like.device}; got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")
    sb, si, sj, sd = t.stride()
    if sd != 1 and t.shape[3] != 1 and t.numel():
        raise ValueError(f"{name} must have contiguous channels; got strides {t.stride()}")
    return _lib.PairTensor(t.data_ptr(), sb, si, sj)


def _out(t: Optional[torch.Tensor], like: torch.Tensor, name: str, dtype: Optional[torch.dtype] = None) -> Optional[int]:
    if t is None:
        return None
    dtype = dtype or like.dtype
    if t.shape != like.shape or t.dtype is not dtype or t.device != like.device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {tuple(like.shape)} {dtype} tensor on {like.device}; got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}")
    return t.data_ptr()


def _gain(weight: torch.Tensor, like: torch.Tensor, name: str = "weight") -> int:
    _kind(weight, name)
    if tuple(weight.shape) != (like.shape[3],) or weight.device != like.device or not weight.is_contiguous():
        raise ValueError(f"{name} must be a contiguous ({like.shape[3]},) tensor on {like.device}; got "
                         f"{tuple(weight.shape)} on {weight.device}")
    return weight.data_ptr()


def _stream(like: torch.Tensor) -> int:
    if like.device.index != torch.cuda.current_device():
        raise ValueError(f"the kernels run on the current device; make {like.device} current (torch.cuda.device)")
    return torch.cuda.current_stream(like.device).cuda_stream


def dropout_desc(keep: int = 65536, seed: int = 0, offset: int = 0, shared: int = _lib.PAIR_SHARED_NONE,
                 origin=(0, 0, 0), device_seed: Optional[torch.Tensor] = None) -> _lib.PairDropoutDesc:
    """The library's record of a dropout: ``keep`` of 65536 values stay; ``device_seed`` is an int64 CUDA tensor
    ``[seed, offset]`` that the kernel reads when it runs."""
    if device_seed is not None:
        if device_seed.dtype is not torch.int64 or device_seed.numel() != 2 or not device_seed.is_cuda or not device_seed.is_contiguous():
            raise ValueError("device_seed must be a contiguous int64 CUDA tensor of two values [seed, offset]")
    return _lib.PairDropoutDesc(seed, offset, keep, None if device_seed is None else device_seed.data_ptr(), shared, *origin)


_NO_DROPOUT = dropout_desc()


def norm_desc(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-5, group: int = 0,
              dropout: Optional[_lib.PairDropoutDesc] = None) -> _lib.PairNormDesc:
    _cuda(x, "update")
    if x.dim() != 4:
        raise ValueError(f"activations must be (B, N_i, N_j, D); got {tuple(x.shape)}")
    kind = _kind(x, "update")
    wkind = kind if weight is None else _kind(weight, "weight")
    return _lib.PairNormDesc(*x.shape, kind, wkind, group, eps, _NO_DROPOUT if dropout is None else dropout)


def add_norm(update: torch.Tensor, residual: Optional[torch.Tensor], weight: Optional[torch.Tensor],
             stream: Optional[torch.Tensor], y: Optional[torch.Tensor], scales: Optional[torch.Tensor] = None, *,
             eps: float = 1e-5, group: int = 0, dropout: Optional[_lib.PairDropoutDesc] = None) -> None:
    """``stream = residual + dropout(update)``; with ``weight``, ``y = rms_norm(stream) * weight``; with ``group``, ``y`` is
    ``float8_e4m3fn`` and ``scales`` holds one fp32 per ``group`` channels.  ``stream`` may be the memory of a contiguous
    ``residual`` or ``update`` itself."""
    desc = norm_desc(update, weight, eps, group, dropout)
    u, r = _view(update, update, "update"), _view(residual, update, "residual")
    w = None if weight is None else _gain(weight, update)
    sptr = None
    if group:
        if scales is None or scales.dtype is not torch.float32 or not scales.is_contiguous() or scales.device != update.device \
                or scales.numel() * group != update.numel():
            raise ValueError(f"scales must be a contiguous float32 tensor with one value per {group} channels")
        sptr = scales.data_ptr()
    rc = _lib.load().pair_sm100_add_norm(C.byref(desc), C.byref(u), C.byref(r), w, _out(stream, update, "stream"),
                                         _out(y, update, "y", torch.float8_e4m3fn if group else None), sptr, _stream(update))
    _lib.check(rc, "pair_sm100_add_norm")


def add_norm_grad_workspace(desc: _lib.PairNormDesc) -> int:
    n = C.c_uint64(0)
    _lib.check(_lib.load().pair_sm100_add_norm_grad_workspace(C.byref(desc), C.byref(n)), "pair_sm100_add_norm_grad_workspace")
    return n.value


def add_norm_grad(stream: torch.Tensor, dy: Optional[torch.Tensor], dz: Optional[torch.Tensor], weight: torch.Tensor,
                  d_stream: Optional[torch.Tensor], d_update: Optional[torch.Tensor], d_weight: Optional[torch.Tensor],
                  workspace: Optional[torch.Tensor], *, eps: float = 1e-5,
                  dropout: Optional[_lib.PairDropoutDesc] = None) -> None:
    """Gradients of :func:`add_norm` with a ``weight``, from the ``stream`` it stored."""
    desc = norm_desc(stream, weight, eps, 0, dropout)
    z, y, g = _view(stream, stream, "stream"), _view(dy, stream, "dy"), _view(dz, stream, "dz")
    wptr = None
    if d_weight is not None:
        if d_weight.dtype is not weight.dtype:
            raise ValueError(f"d_weight must be {weight.dtype}; got {d_weight.dtype}")
        wptr = _gain(d_weight, stream, "d_weight")
        need = add_norm_grad_workspace(desc)
        if workspace is None or workspace.numel() * workspace.element_size() < need or workspace.device != stream.device:
            raise ValueError(f"workspace must be a tensor of at least {need} bytes on {stream.device}")
    rc = _lib.load().pair_sm100_add_norm_grad(C.byref(desc), C.byref(z), C.byref(y), C.byref(g), _gain(weight, stream),
                                              _out(d_stream, stream, "d_stream"), _out(d_update, stream, "d_update"), wptr,
                                              None if workspace is None else workspace.data_ptr(), _stream(stream))
    _lib.check(rc, "pair_sm100_add_norm_grad")


def embed_desc(index: torch.Tensor, table: torch.Tensor, dtype: torch.dtype, scale: float) -> _lib.PairEmbedDesc:
    _cuda(index, "index")
    _cuda(table, "table")
    if index.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"index must be int32 or int64; got {index.dtype}")
    if table.dim() != 2 or table.device != index.device:
        raise ValueError(f"table must be (V, D) on {index.device}; got {tuple(table.shape)} on {table.device}")
    if dtype not in DTYPES:
        raise ValueError(f"the embedding's type must be bfloat16, float16 or float32; got {dtype}")
    rows, d = table.shape
    return _lib.PairEmbedDesc(index.numel(), d, rows, 32 if index.dtype is torch.int32 else 64, DTYPES[dtype],
                              _kind(table, "table"), scale)


def _flat(t: torch.Tensor, name: str, shape, dtype: torch.dtype, device) -> int:
    if tuple(t.shape) != tuple(shape) or t.dtype is not dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {tuple(shape)} {dtype} tensor on {device}; got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}, strides {t.stride()}")
    return t.data_ptr()


def embed(index: torch.Tensor, table: torch.Tensor, base: Optional[torch.Tensor], out: torch.Tensor, *,
          scale: float = 1.0) -> None:
    """``out = base + scale * table[index]``; an index outside the table adds nothing.  ``out`` may be ``base``."""
    desc = embed_desc(index, table, out.dtype, scale)
    dev, shape = index.device, (*index.shape, table.shape[1])
    iptr = _flat(index, "index", index.shape, index.dtype, dev)
    tptr = _flat(table, "table", table.shape, table.dtype, dev)
    bptr = None if base is None else _flat(base, "base", shape, out.dtype, dev)
    rc = _lib.load().pair_sm100_embed(C.byref(desc), iptr, tptr, bptr, _flat(out, "out", shape, out.dtype, dev), _stream(index))
    _lib.check(rc, "pair_sm100_embed")


def embed_grad_workspace(desc: _lib.PairEmbedDesc) -> int:
    n = C.c_uint64(0)
    _lib.check(_lib.load().pair_sm100_embed_grad_workspace(C.byref(desc), C.byref(n)), "pair_sm100_embed_grad_workspace")
    return n.value


def embed_grad(index: torch.Tensor, d_out: torch.Tensor, d_table: torch.Tensor, workspace: Optional[torch.Tensor], *,
               scale: float = 1.0) -> None:
    """``d_table[v] = scale * sum(d_out[index == v])``, summed in a fixed order."""
    desc = embed_desc(index, d_table, d_out.dtype, scale)
    dev = index.device
    need = embed_grad_workspace(desc)
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need or workspace.device != dev):
        raise ValueError(f"workspace must be a tensor of at least {need} bytes on {dev}")
    rc = _lib.load().pair_sm100_embed_grad(
        C.byref(desc), _flat(index, "index", index.shape, index.dtype, dev),
        _flat(d_out, "d_out", (*index.shape, d_table.shape[1]), d_out.dtype, dev),
        _flat(d_table, "d_table", d_table.shape, d_table.dtype, dev),
        None if workspace is None else workspace.data_ptr(), _stream(index))
    _lib.check(rc, "pair_sm100_embed_grad")
