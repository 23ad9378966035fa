"""Per-kernel Python entry points of the pair-stream operators, over the C ABI of ``include/pair_stream_sm100.h``.

As in :mod:`fold_cp_ops_b200.kernels`, each function checks types and layouts, passes device pointers and the
current CUDA stream to the library and writes into tensors that the caller provides (the ``*_workspace`` functions say
how many bytes of scratch to provide).  :mod:`fold_cp_ops_b200.workflows.pair_stream` allocates and differentiates.

Activations are ``(B, N_i, N_j, D)`` tensors of any strides whose channels are contiguous; outputs are contiguous.

The ``launch_*`` functions are the calls themselves, for callers that have checked their tensors already.  A call on
a small tensor is host time, so the library's records are packed with :mod:`struct` (about 1 us) instead of being
built field by field (4 us); a CPU test holds the formats to the header's layout.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
from typing import Optional, Sequence

import torch

from . import _lib

DTYPES = {torch.bfloat16: _lib.PAIR_BF16, torch.float16: _lib.PAIR_FP16, torch.float32: _lib.PAIR_FP32}

#: fields of a ``pair_dropout_t``: seed, offset, keep, device_seed, shared, origin b, i, j
NO_DROPOUT = (0, 0, 65536, 0, _lib.PAIR_SHARED_NONE, 0, 0, 0)

_pack_norm = struct.Struct("@7if QIIP4i").pack    # pair_norm_desc_t
_pack_tensor = struct.Struct("@P3q").pack         # pair_tensor_t
_pack_embed = struct.Struct("@q5if").pack         # pair_embed_desc_t
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


# ---------------------------------------------------------------------------------------------
# the calls
# ---------------------------------------------------------------------------------------------
def _view(t: Optional[torch.Tensor]):
    if t is None:
        return None
    s = t.stride()
    return _pack_tensor(t.data_ptr(), s[0], s[1], s[2])


def _at(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def launch_add_norm(update, residual, weight, stream, y, scales, eps: float, group: int, dropout) -> None:
    kind = DTYPES[update.dtype]
    wkind = kind if weight is None else DTYPES[weight.dtype]
    rc = _lib.load().pair_sm100_add_norm(_pack_norm(*update.shape, kind, wkind, group, eps, *dropout), _view(update),
                                         _view(residual), _at(weight), _at(stream), _at(y), _at(scales),
                                         _raw_stream(update.device.index))
    if rc:
        _lib.check(rc, "pair_sm100_add_norm")


def launch_add_norm_grad(stream, dy, dz, weight, d_stream, d_update, d_weight, workspace, eps: float, dropout) -> None:
    desc = _pack_norm(*stream.shape, DTYPES[stream.dtype], DTYPES[weight.dtype], 0, eps, *dropout)
    rc = _lib.load().pair_sm100_add_norm_grad(desc, _view(stream), _view(dy), _view(dz), weight.data_ptr(), _at(d_stream),
                                              _at(d_update), _at(d_weight), _at(workspace), _raw_stream(stream.device.index))
    if rc:
        _lib.check(rc, "pair_sm100_add_norm_grad")


def launch_embed(index, table, base, out, scale: float) -> None:
    rows, d = table.shape
    desc = _pack_embed(index.numel(), d, rows, 32 if index.dtype is torch.int32 else 64, DTYPES[out.dtype],
                       DTYPES[table.dtype], scale)
    rc = _lib.load().pair_sm100_embed(desc, index.data_ptr(), table.data_ptr(), _at(base), out.data_ptr(),
                                      _raw_stream(index.device.index))
    if rc:
        _lib.check(rc, "pair_sm100_embed")


def launch_embed_grad(index, d_out, d_table, workspace, scale: float) -> None:
    rows, d = d_table.shape
    desc = _pack_embed(index.numel(), d, rows, 32 if index.dtype is torch.int32 else 64, DTYPES[d_out.dtype],
                       DTYPES[d_table.dtype], scale)
    rc = _lib.load().pair_sm100_embed_grad(desc, index.data_ptr(), d_out.data_ptr(), d_table.data_ptr(), _at(workspace),
                                           _raw_stream(index.device.index))
    if rc:
        _lib.check(rc, "pair_sm100_embed_grad")


@functools.lru_cache(maxsize=1024)
def _norm_grad_bytes(device: int, rows: int, d: int) -> int:
    n = C.c_uint64(0)
    with torch.cuda.device(device):
        desc = _pack_norm(1, 1, rows, d, _lib.PAIR_BF16, _lib.PAIR_BF16, 0, 1.0, *NO_DROPOUT)
        _lib.check(_lib.load().pair_sm100_add_norm_grad_workspace(desc, C.byref(n)), "pair_sm100_add_norm_grad_workspace")
    return n.value


@functools.lru_cache(maxsize=1024)
def _embed_grad_bytes(device: int, tokens: int, rows: int, d: int) -> int:
    n = C.c_uint64(0)
    with torch.cuda.device(device):
        desc = _pack_embed(tokens, d, rows, 64, _lib.PAIR_BF16, _lib.PAIR_BF16, 1.0)
        _lib.check(_lib.load().pair_sm100_embed_grad_workspace(desc, C.byref(n)), "pair_sm100_embed_grad_workspace")
    return n.value


# ---------------------------------------------------------------------------------------------
# the checked entry points
# ---------------------------------------------------------------------------------------------
def _activation(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor; the pair-stream kernels have no CPU path")
    if t.dtype not in DTYPES:
        raise ValueError(f"{name} must be bfloat16, float16 or float32; got {t.dtype}")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"the kernels run on the current device; make {t.device} current (torch.cuda.device)")


def _pair(t: Optional[torch.Tensor], like: torch.Tensor, name: str) -> None:
    if t is None:
        return
    if t.dim() != 4 or t.shape != like.shape or t.dtype is not like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be (B, N_i, N_j, D) like {tuple(like.shape)} {like.dtype} on {like.device}; got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    if t.stride(3) != 1 and t.shape[3] != 1 and t.numel():
        raise ValueError(f"{name} must have contiguous channels; got strides {t.stride()}")


def _contiguous(t: Optional[torch.Tensor], shape: Sequence[int], dtype: torch.dtype, device, name: str) -> None:
    if t is not None and (tuple(t.shape) != tuple(shape) or t.dtype is not dtype or t.device != device or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {tuple(shape)} {dtype} tensor on {device}; got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}, strides {t.stride()}")


def _gain(weight: torch.Tensor, like: torch.Tensor) -> None:
    if weight.dtype not in DTYPES:
        raise ValueError(f"weight must be bfloat16, float16 or float32; got {weight.dtype}")
    _contiguous(weight, like.shape[3:], weight.dtype, like.device, "weight")


def _scratch(workspace: Optional[torch.Tensor], need: int, device) -> None:
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need or workspace.device != device):
        raise ValueError(f"workspace must be a tensor of at least {need} bytes on {device}")


def dropout_record(keep: int = 65536, seed: int = 0, offset: int = 0, shared: int = _lib.PAIR_SHARED_NONE,
                   origin=(0, 0, 0), device_seed: Optional[torch.Tensor] = None) -> tuple:
    """The library's record of a dropout: ``keep`` of 65536 values stay; ``device_seed`` is an int64 CUDA tensor
    ``[seed, offset]`` that the kernel reads when it runs."""
    if device_seed is not None and (device_seed.dtype is not torch.int64 or device_seed.numel() != 2
                                    or not device_seed.is_cuda or not device_seed.is_contiguous()):
        raise ValueError("device_seed must be a contiguous int64 CUDA tensor of two values [seed, offset]")
    return (seed, offset, keep, 0 if device_seed is None else device_seed.data_ptr(), shared, *origin)


def add_norm(update: torch.Tensor, residual: Optional[torch.Tensor], weight: Optional[torch.Tensor],
             stream: Optional[torch.Tensor], y: Optional[torch.Tensor], scales: Optional[torch.Tensor] = None, *,
             eps: float = 1e-5, group: int = 0, dropout: tuple = NO_DROPOUT) -> None:
    """``stream = residual + dropout(update)``; with ``weight``, ``y = rms_norm(stream) * weight``; with ``group``, ``y`` is
    ``float8_e4m3fn`` and ``scales`` holds one fp32 per ``group`` channels.  ``stream`` may be the memory of a contiguous
    ``residual`` or ``update`` itself."""
    _activation(update, "update")
    _pair(update, update, "update")
    _pair(residual, update, "residual")
    if weight is not None:
        _gain(weight, update)
    _contiguous(stream, update.shape, update.dtype, update.device, "stream")
    _contiguous(y, update.shape, torch.float8_e4m3fn if group else update.dtype, update.device, "y")
    if group and (scales is None or scales.dtype is not torch.float32 or not scales.is_contiguous()
                  or scales.device != update.device or scales.numel() * group != update.numel()):
        raise ValueError(f"scales must be a contiguous float32 tensor with one value per {group} channels")
    launch_add_norm(update, residual, weight, stream, y, scales, eps, group, dropout)


def add_norm_grad_workspace(stream: torch.Tensor) -> int:
    """Bytes of workspace that :func:`add_norm_grad` needs for a gain's gradient over these rows."""
    d = stream.shape[-1]
    return _norm_grad_bytes(stream.device.index, stream.numel() // d, d)


def add_norm_grad(stream: torch.Tensor, dy: Optional[torch.Tensor], dz: Optional[torch.Tensor], weight: torch.Tensor,
                  d_stream: Optional[torch.Tensor], d_update: Optional[torch.Tensor], d_weight: Optional[torch.Tensor],
                  workspace: Optional[torch.Tensor], *, eps: float = 1e-5, dropout: tuple = NO_DROPOUT) -> None:
    """Gradients of :func:`add_norm` with a ``weight``, from the ``stream`` it stored."""
    _activation(stream, "stream")
    for t, name in ((stream, "stream"), (dy, "dy"), (dz, "dz")):
        _pair(t, stream, name)
    _gain(weight, stream)
    for t, name in ((d_stream, "d_stream"), (d_update, "d_update")):
        _contiguous(t, stream.shape, stream.dtype, stream.device, name)
    if d_weight is not None:
        _contiguous(d_weight, weight.shape, weight.dtype, weight.device, "d_weight")
        _scratch(workspace, add_norm_grad_workspace(stream), stream.device)
    launch_add_norm_grad(stream, dy, dz, weight, d_stream, d_update, d_weight, workspace, eps, dropout)


def _embedding(index: torch.Tensor, table: torch.Tensor, out: torch.Tensor, table_name: str, out_name: str) -> None:
    _activation(out, out_name)
    _activation(table, table_name)
    if index.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"index must be int32 or int64; got {index.dtype}")
    if table.dim() != 2:
        raise ValueError(f"{table_name} must be (V, D); got {tuple(table.shape)}")
    _contiguous(index, index.shape, index.dtype, out.device, "index")
    _contiguous(table, table.shape, table.dtype, out.device, table_name)
    _contiguous(out, (*index.shape, table.shape[1]), out.dtype, out.device, out_name)


def embed(index: torch.Tensor, table: torch.Tensor, base: Optional[torch.Tensor], out: torch.Tensor, *,
          scale: float = 1.0) -> None:
    """``out = base + scale * table[index]``; an index outside the table adds nothing.  ``out`` may be ``base``."""
    _embedding(index, table, out, "table", "out")
    _contiguous(base, out.shape, out.dtype, out.device, "base")
    launch_embed(index, table, base, out, scale)


def embed_grad_workspace(index: torch.Tensor, table: torch.Tensor) -> int:
    """Bytes of workspace that :func:`embed_grad` needs."""
    return _embed_grad_bytes(table.device.index, index.numel(), *table.shape)


def embed_grad(index: torch.Tensor, d_out: torch.Tensor, d_table: torch.Tensor, workspace: Optional[torch.Tensor], *,
               scale: float = 1.0) -> None:
    """``d_table[v] = scale * sum(d_out[index == v])``, summed in a fixed order."""
    _embedding(index, d_table, d_out, "d_table", "d_out")
    _scratch(workspace, embed_grad_workspace(index, d_table), index.device)
    launch_embed_grad(index, d_out, d_table, workspace, scale)
