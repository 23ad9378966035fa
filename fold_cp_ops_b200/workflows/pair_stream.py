"""The pair stream around the triangle update: what makes it, what is added to it, what reads it.

A pair stack keeps one representation ``z`` of shape ``(B, N_i, N_j, D)``.  The triangle update (this package's other
operators) computes an update of it; the functions here are the rest of the stream, each one pass over HBM:

* :func:`dropout_add` -- ``z = residual + dropout(update)``;
* :func:`add_rms_norm` -- the same, and the root-mean-square norm of ``z`` that the next block reads;
* :func:`add_rms_norm_fp8` -- the same with the norm in e4m3 and fp32 scales, for an 8-bit product;
* :func:`pair_embedding` -- ``base + scale * table[index]``: position or distance bins, residue types.

All but the e4m3 form have gradients (once differentiable).  Statistics and sums are fp32 or wider whatever the tensors'
type; ``z`` is rounded once, to the activations' type, and the norm reads ``z`` as it is stored.

Dropout (:class:`PairDropout`) stores no mask: element ``(b, i, j, c)`` of the WHOLE grid is kept by a counter-based
generator of exactly that position, so the gradient draws the mask again, and ranks that hold different blocks of a
context-parallel grid draw the same mask as one GPU would.

Tensors may be DTensors sharded over batch and token dims, as the distributed triangle update takes them: the blocks'
positions are then taken from the placements.  Gradients are for plain tensors only.  Inputs need contiguous channels
(others are copied); other strides -- a transposed view, a block of a larger tensor, a broadcast axis -- are read in place.
There is no CPU path.
"""
from __future__ import annotations

import math
from dataclasses import dataclass, replace
from typing import Optional, Sequence, Tuple, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import _lib
from .. import pair_kernels as PK
from ..distributed.dtensor_adapter import _dtensor_mesh_placements, _is_dtensor, _rowmaj_stride, _shards

__all__ = ["PairDropout", "dropout_add", "add_rms_norm", "add_rms_norm_fp8", "pair_embedding", "pair_block_origin"]

_SHARED = {None: _lib.PAIR_SHARED_NONE, "rows": _lib.PAIR_SHARED_ROWS, "columns": _lib.PAIR_SHARED_COLUMNS}
_BYTE = torch.uint8
_PLAIN = frozenset((Tensor, torch.nn.Parameter, type(None)))
_NO_DTENSOR_GRADIENT = "gradients through DTensors are not supported: pass the local blocks, with PairDropout.origin"


@dataclass(frozen=True)
class PairDropout:
    """A dropout of pair tensors whose mask is a function of its arguments alone.

    ``p``: probability of being dropped, in multiples of 2^-16 (the nearest is taken); kept elements are multiplied by the
    exact reciprocal of the probability of being kept.  ``seed`` (64 bits) and ``offset`` (32 bits) name the mask: give every
    layer and step its own pair.  For captured graphs ``seed`` may be a CUDA tensor of two int64 values ``[seed, offset]``
    that is read when the kernel runs (``offset`` is then ignored here); it must keep its values until the gradient is computed.
    ``shared``: ``"rows"`` -- one mask for all rows ``i``; ``"columns"`` -- one for all columns ``j``; ``None`` -- every
    element its own.  ``origin``: the ``(b, i, j)`` of the tensor's first element in the whole grid, where the tensor is one
    rank's block (DTensors know theirs)."""

    p: float
    seed: Union[int, Tensor] = 0
    offset: int = 0
    shared: Optional[str] = None
    origin: Tuple[int, int, int] = (0, 0, 0)

    def __post_init__(self):
        if not 0.0 <= self.p <= 1.0:
            raise ValueError(f"p must be in [0, 1]; got {self.p}")
        if self.shared not in _SHARED:
            raise ValueError(f"shared must be None, 'rows' or 'columns'; got {self.shared!r}")
        if isinstance(self.seed, Tensor):
            if self.seed.dtype is not torch.int64 or self.seed.numel() != 2 or not self.seed.is_cuda or not self.seed.is_contiguous():
                raise ValueError("seed must be an int or a contiguous int64 CUDA tensor of two values [seed, offset]")
        elif not 0 <= self.seed < 1 << 64:
            raise ValueError(f"seed must fit 64 bits unsigned; got {self.seed}")
        if not 0 <= self.offset < 1 << 32:
            raise ValueError(f"offset must fit 32 bits unsigned; got {self.offset}")
        if len(self.origin) != 3 or not all(0 <= o < 1 << 31 for o in self.origin):
            raise ValueError(f"origin must be three coordinates (b, i, j) >= 0; got {self.origin}")

    @property
    def keep(self) -> int:
        """How many of 65536 values are kept."""
        return math.floor((1.0 - self.p) * 65536.0 + 0.5)

    def _record(self) -> tuple:
        on_device = isinstance(self.seed, Tensor)
        return PK.dropout_record(self.keep, 0 if on_device else self.seed, self.offset, _SHARED[self.shared], self.origin,
                                 self.seed if on_device else None)


def pair_block_origin(x) -> Tuple[int, int, int]:
    """``(b, i, j)`` of this rank's first element of a pair DTensor in the whole grid."""
    from torch.distributed.tensor._utils import compute_local_shape_and_global_offset

    mesh, placements = _dtensor_mesh_placements(x)
    _, offset = compute_local_shape_and_global_offset(x.shape, mesh, placements)
    return tuple(int(o) for o in offset[:3])


# ---------------------------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------------------------
def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _locals_of(names: Sequence[str], tensors: Sequence[Optional[Tensor]]):
    """The ranks' local blocks of DTensors that are sharded alike, and their :class:`_Wrap` (``None`` where all are plain)."""
    if all(type(t) in _PLAIN for t in tensors):
        return tensors, None
    given = [(n, t) for n, t in zip(names, tensors) if t is not None]
    if not any(_is_dtensor(t) for _, t in given):
        return tensors, None
    if not all(_is_dtensor(t) for _, t in given):
        raise ValueError(f"{', '.join(n for n, _ in given)} must be DTensors of the same placements or all plain tensors")
    if _needs_grad(*[t for _, t in given]):
        raise ValueError(_NO_DTENSOR_GRADIENT)
    first, x = given[0]
    mesh, placements = _dtensor_mesh_placements(x)
    tokens = 3 if first != "index" else x.dim()
    if first != "index" and x.dim() != 4:
        raise ValueError(f"{first} as a DTensor must be (B, N_i, N_j, D); got {tuple(x.shape)}")
    for n, t in given[1:]:
        if _dtensor_mesh_placements(t) != (mesh, placements):
            raise ValueError(f"{n} must have the mesh and placements of {first}: {placements}")
    if any(dim >= tokens for _, dim in _shards(placements)):
        raise ValueError(f"the channels must be whole on every rank, but {placements} shard them")
    if any(p.is_partial() for p in placements):
        raise ValueError(f"{first} holds partial sums ({placements}): reduce it first")
    return [None if t is None else t.to_local() for t in tensors], _Wrap(mesh, placements, x, tokens)


class _Wrap:
    """Makes local results DTensors again."""

    def __init__(self, mesh, placements, like, tokens: int):
        self.mesh, self.placements, self.like, self.tokens = mesh, placements, like, tuple(like.shape[:tokens])

    def __call__(self, local: Tensor):
        from torch.distributed.tensor import DTensor

        shape = torch.Size((*self.tokens, *local.shape[len(self.tokens):]))
        return DTensor.from_local(local, self.mesh, self.placements, run_check=False, shape=shape, stride=_rowmaj_stride(shape))


def _placed(dropout: Optional[PairDropout], wrap: Optional[_Wrap]) -> Optional[PairDropout]:
    """``dropout`` at the position of this rank's block, or ``None`` where it keeps everything."""
    if dropout is not None and not isinstance(dropout, PairDropout):
        raise TypeError(f"dropout must be a PairDropout or None; got {type(dropout).__name__}")
    if dropout is None or dropout.keep == 65536:
        return None
    if wrap is None:
        return dropout
    return replace(dropout, origin=tuple(o + at for o, at in zip(dropout.origin, pair_block_origin(wrap.like))))


def _span(t: Tensor) -> Tuple[int, int]:
    """First byte and end of the memory a tensor reaches."""
    at = t.data_ptr()
    return at, at + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _check_overlap(out: Tensor, t: Optional[Tensor], name: str) -> None:
    if t is None or out.numel() == 0:
        return
    (a, b), (c, d) = _span(out), _span(t)
    if a < d and c < b and not (a == c and t.is_contiguous()):
        raise ValueError(f"out overlaps {name} without being it")


def _as_pair(t: Optional[Tensor]) -> Optional[Tensor]:
    """A four-dimensional view with contiguous channels (a copy where they are not)."""
    if t is None:
        return None
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        t = t.contiguous()
    return t if t.dim() == 4 else t[(None,) * (4 - t.dim())]


def _aligned(t: Optional[Tensor]) -> Optional[Tensor]:
    """``t``, or a copy of it where its rows do not start on 16-byte boundaries."""
    if t is None:
        return None
    unit = 16 // t.element_size()
    if t.data_ptr() % 16 == 0 and all(s % unit == 0 for s in t.stride()[:-1]) and (t.stride(-1) == 1 or t.shape[-1] == 1):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check_pair(update: Tensor, residual: Optional[Tensor]) -> None:
    if not isinstance(update, Tensor):
        raise TypeError(f"update must be a tensor; got {type(update).__name__}")
    if not update.is_cuda:
        raise ValueError("update must be a CUDA tensor; the pair-stream kernels have no CPU path")
    if update.dtype not in PK.DTYPES:
        raise ValueError(f"update must be bfloat16, float16 or float32; got {update.dtype}")
    if not 1 <= update.dim() <= 4:
        raise ValueError(f"update must have one to four dims, (B, N_i, N_j, D) or its last ones; got {tuple(update.shape)}")
    if not 1 <= update.shape[-1] <= _lib.PAIR_MAX_WIDTH:
        raise ValueError(f"the width D must be in [1, {_lib.PAIR_MAX_WIDTH}]; got {update.shape[-1]}")
    if update.numel() // update.shape[-1] >= 1 << 31:
        raise ValueError(f"at most 2^31 - 1 rows in one call; got {tuple(update.shape)}")
    if residual is not None and (residual.shape != update.shape or residual.dtype is not update.dtype
                                 or residual.device != update.device):
        raise ValueError(f"residual must be {tuple(update.shape)} {update.dtype} on {update.device} like update; got "
                         f"{tuple(residual.shape)} {residual.dtype} on {residual.device}")


def _check_weight(weight: Tensor, update: Tensor, eps: float) -> None:
    if tuple(weight.shape) != (update.shape[-1],) or weight.dtype not in PK.DTYPES or weight.device != update.device:
        raise ValueError(f"weight must be a ({update.shape[-1]},) bfloat16, float16 or float32 tensor on {update.device}; got "
                         f"{tuple(weight.shape)} {weight.dtype} on {weight.device}")
    if not 1.1754944e-38 <= eps < 3.4e38:
        raise ValueError(f"eps must be a normal float32 number > 0; got {eps}")


def _elsewhere(device: torch.device):
    """A context that makes ``device`` current, or ``None`` where it is."""
    return None if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _new(like: Tensor, dtype: Optional[torch.dtype] = None) -> Tensor:
    return torch.empty_like(like, dtype=dtype, memory_format=torch.contiguous_format)


# ---------------------------------------------------------------------------------------------
# the addition and the norm
# ---------------------------------------------------------------------------------------------
# The _run_* functions take checked tensors, allocate what they return and launch on the current stream of the tensors'
# device.  A dropout comes as the library's record.
def _run_add(update, residual, record, out=None) -> Tensor:
    elsewhere = _elsewhere(update.device)
    if elsewhere is not None:
        with elsewhere:
            return _run_add(update, residual, record, out)
    z = _new(update) if out is None else out
    PK.launch_add_norm(_as_pair(update), _as_pair(residual), None, _as_pair(z), None, None, 1.0, 0, record)
    return z


def _run_norm(update, residual, weight, eps, record, group=0):
    elsewhere = _elsewhere(update.device)
    if elsewhere is not None:
        with elsewhere:
            return _run_norm(update, residual, weight, eps, record, group)
    # without a residual and a dropout the stream is the update itself
    z = None if residual is None and record is PK.NO_DROPOUT else _new(update)
    y, scales = _new(update, torch.float8_e4m3fn if group else None), None
    if group:
        scales = torch.empty((*update.shape[:-1], update.shape[-1] // group), dtype=torch.float32, device=update.device)
    PK.launch_add_norm(_as_pair(update), _as_pair(residual), weight.contiguous(), _as_pair(z), _as_pair(y), scales, eps, group,
                       record)
    return y, z, scales


def _run_norm_grad(z, dy, dz, weight, eps, record, need_u, need_r, need_w):
    """``(d_update, d_residual, d_weight)``; without a dropout the first two are one tensor."""
    elsewhere = _elsewhere(z.device)
    if elsewhere is not None:
        with elsewhere:
            return _run_norm_grad(z, dy, dz, weight, eps, record, need_u, need_r, need_w)
    dropped = record is not PK.NO_DROPOUT
    du = _new(z) if need_u and (dropped or not need_r) else None
    dr = _new(z) if need_r else None
    dw = workspace = None
    if need_w:
        dw = _new(weight)
        workspace = torch.empty(PK.add_norm_grad_workspace(z), dtype=_BYTE, device=z.device)
    PK.launch_add_norm_grad(_as_pair(z), _as_pair(dy), _as_pair(dz), weight.contiguous(), _as_pair(dr), _as_pair(du), dw,
                            workspace, eps, record)
    return dr if need_u and du is None else du, dr, dw


def _seed_of(dropout: Optional[PairDropout]) -> Optional[Tensor]:
    """A device seed, to be saved for the gradient: a change of its values until then is an error."""
    return dropout.seed if dropout is not None and isinstance(dropout.seed, Tensor) else None


def _record_of(dropout: Optional[PairDropout]) -> tuple:
    return PK.NO_DROPOUT if dropout is None else dropout._record()


class _Once(torch.autograd.Function):
    """A function without a second derivative.  ``once_differentiable`` costs host time and matters only where a graph of
    the gradient is being made."""

    @classmethod
    def backward(cls, ctx, *grads):
        return cls.marked(ctx, *grads) if torch.is_grad_enabled() else cls.gradient(ctx, *grads)

    def __init_subclass__(cls):
        cls.marked = staticmethod(once_differentiable(cls.gradient))


class _DropoutAdd(_Once):
    @staticmethod
    def forward(ctx, update, residual, dropout):
        ctx.set_materialize_grads(False)
        ctx.record = _record_of(dropout)
        ctx.save_for_backward(_seed_of(dropout))
        return _run_add(update, residual, ctx.record)

    @staticmethod
    def gradient(ctx, dz):
        if dz is None:
            return None, None, None
        ctx.saved_tensors  # raises where the seed's values were changed
        need_u, need_r, _ = ctx.needs_input_grad
        du = None
        if need_u:
            du = dz if ctx.record is PK.NO_DROPOUT else _run_add(dz, None, ctx.record)
        return du, dz if need_r else None, None


class _AddRmsNorm(_Once):
    @staticmethod
    def forward(ctx, update, residual, weight, eps, dropout):
        ctx.set_materialize_grads(False)
        record = _record_of(dropout)
        y, z, _ = _run_norm(update, residual, weight, eps, record)
        if z is None:
            z = update.view_as(update)
        ctx.args = eps, record
        ctx.save_for_backward(z, weight, _seed_of(dropout))
        return y, z

    @staticmethod
    def gradient(ctx, dy, dz):
        if dy is None and dz is None:
            return None, None, None, None, None
        z, weight, _ = ctx.saved_tensors
        return (*_run_norm_grad(z, dy, dz, weight, *ctx.args, *ctx.needs_input_grad[:3]), None, None)


def dropout_add(update: Tensor, residual: Optional[Tensor] = None, dropout: Optional[PairDropout] = None, *,
                out: Optional[Tensor] = None) -> Tensor:
    """``residual + dropout(update)`` in the tensors' type (bfloat16, float16 or float32), added in fp32.

    ``update`` and ``residual``: ``(B, N_i, N_j, D)`` or its last dims, of one shape, type and device, any strides.
    ``residual=None`` is a plain dropout.  ``out`` (contiguous; no gradients) may be ``residual`` or ``update`` itself: the
    stream is then updated in place.  Dropped elements become 0 whatever they were.  Raises ``ValueError`` for anything
    else, ``TypeError`` for a ``dropout`` that is no :class:`PairDropout`."""
    given = out
    (update, residual, out), wrap = _locals_of(("update", "residual", "out"), (update, residual, out))
    dropout = _placed(dropout, wrap)
    _check_pair(update, residual)
    if out is not None:
        if _needs_grad(update, residual, out):
            raise ValueError("out= has no gradient: leave it out, or run under torch.no_grad()")
        if out.shape != update.shape or out.dtype is not update.dtype or out.device != update.device or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {tuple(update.shape)} {update.dtype} tensor on {update.device}")
        _check_overlap(out, update, "update")
        _check_overlap(out, residual, "residual")
    elif _needs_grad(update, residual):
        return _DropoutAdd.apply(update, residual, dropout)
    z = _run_add(update, residual, _record_of(dropout), out)
    if given is not None:
        return given
    return z if wrap is None else wrap(z)


def add_rms_norm(update: Tensor, residual: Optional[Tensor], weight: Tensor, *, eps: float = 1e-5,
                 dropout: Optional[PairDropout] = None) -> Tuple[Tensor, Tensor]:
    """``(y, z)``: ``z = residual + dropout(update)`` and ``y = z / sqrt(mean(z^2) + eps) * weight`` over the channels.

    Tensors as in :func:`dropout_add`; ``weight`` is ``(D,)`` in any of the three types and gets its gradient in its own.
    ``residual=None`` takes the norm of ``dropout(update)``; without a dropout too, ``z`` is ``update`` itself.  ``D`` is at
    most 8192."""
    (update, residual), wrap = _locals_of(("update", "residual"), (update, residual))
    dropout = _placed(dropout, wrap)
    _check_pair(update, residual)
    _check_weight(weight, update, eps)
    if _needs_grad(update, residual, weight):
        if wrap is not None:
            raise ValueError(_NO_DTENSOR_GRADIENT)
        return _AddRmsNorm.apply(update, residual, weight, eps, dropout)
    y, z, _ = _run_norm(update, residual, weight, eps, _record_of(dropout))
    z = update if z is None else z
    return (y, z) if wrap is None else (wrap(y), wrap(z))


def add_rms_norm_fp8(update: Tensor, residual: Optional[Tensor], weight: Tensor, *, eps: float = 1e-5,
                     group: Optional[int] = 128, dropout: Optional[PairDropout] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """``(q, scales, z)``: :func:`add_rms_norm` with ``y`` in ``float8_e4m3fn``, ``y ~ q * scales`` per ``group`` channels.

    ``group`` is 32, 64 or 128 (dividing ``D``), or ``None`` for one scale per row; ``scales`` is fp32,
    ``(..., D / group)``: the group's largest ``|y|`` / 448, and 1 for a group of zeros.  ``y`` is scaled in fp32 and rounded
    once, to e4m3.  For inference: refuses inputs that require gradients."""
    (update, residual), wrap = _locals_of(("update", "residual"), (update, residual))
    dropout = _placed(dropout, wrap)
    _check_pair(update, residual)
    _check_weight(weight, update, eps)
    width = update.shape[-1]
    if group is not None and (group not in (32, 64, 128) or width % group != 0):
        raise ValueError(f"group must be 32, 64 or 128 and divide D={width}, or None for one scale per row; got {group}")
    if _needs_grad(update, residual, weight):
        raise ValueError("the e4m3 form has no gradient: run it under torch.no_grad()")
    if group is not None:  # lanes reduce a group's octs: rows have to start on 16-byte boundaries
        update, residual = _aligned(update), _aligned(residual)
    y, z, scales = _run_norm(update, residual, weight, eps, _record_of(dropout), group or width)
    z = update if z is None else z
    return (y, scales, z) if wrap is None else (wrap(y), wrap(scales), wrap(z))


# ---------------------------------------------------------------------------------------------
# the embedding
# ---------------------------------------------------------------------------------------------
def _run_embed(index, table, base, scale, dtype) -> Tensor:
    elsewhere = _elsewhere(index.device)
    if elsewhere is not None:
        with elsewhere:
            return _run_embed(index, table, base, scale, dtype)
    out = torch.empty((*index.shape, table.shape[1]), dtype=dtype, device=index.device)
    PK.launch_embed(index, table.contiguous(), None if base is None else base.contiguous(), out, scale)
    return out


def _run_embed_grad(index, d_out, rows, table_dtype, scale) -> Tensor:
    elsewhere = _elsewhere(index.device)
    if elsewhere is not None:
        with elsewhere:
            return _run_embed_grad(index, d_out, rows, table_dtype, scale)
    d_table = torch.empty((rows, d_out.shape[-1]), dtype=table_dtype, device=index.device)
    workspace = torch.empty(PK.embed_grad_workspace(index, d_table), dtype=_BYTE, device=index.device)
    PK.launch_embed_grad(index, d_out.contiguous(), d_table, workspace, scale)
    return d_table


class _PairEmbedding(_Once):
    @staticmethod
    def forward(ctx, index, table, base, scale, dtype):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(index)
        ctx.args = table.shape[0], table.dtype, scale
        return _run_embed(index, table, base, scale, dtype)

    @staticmethod
    def gradient(ctx, d_out):
        if d_out is None:
            return None, None, None, None, None
        (index,) = ctx.saved_tensors
        d_table = _run_embed_grad(index, d_out, *ctx.args) if ctx.needs_input_grad[1] else None
        return None, d_table, d_out if ctx.needs_input_grad[2] else None, None, None


def pair_embedding(index: Tensor, table: Tensor, *, scale: float = 1.0, base: Optional[Tensor] = None,
                   dtype: Optional[torch.dtype] = None) -> Tensor:
    """``base + scale * table[index]``: an embedding lookup into the pair stream, ``(*index.shape, D)``.

    ``index``: int32 or int64, any shape; an entry outside ``[0, V)`` (``-1`` for padding) adds nothing and gets no gradient.
    ``table``: ``(V, D)`` in bfloat16, float16 or float32; its gradient comes in its type, summed in at least fp32 over
    tokens sorted by index, in a fixed order (the same bits every time).  ``base``: what the embedding is added to, or
    ``None``; the result has its type, else ``dtype``, else the table's.  ``index`` and ``base`` may be DTensors sharded
    alike."""
    (index, base), wrap = _locals_of(("index", "base"), (index, base))
    if not isinstance(index, Tensor) or index.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"index must be an int32 or int64 tensor; got {getattr(index, 'dtype', type(index).__name__)}")
    if not index.is_cuda:
        raise ValueError("index must be a CUDA tensor; the pair-stream kernels have no CPU path")
    if table.dim() != 2 or table.shape[0] < 1 or table.dtype not in PK.DTYPES or table.device != index.device:
        raise ValueError(f"table must be a (V, D) bfloat16, float16 or float32 tensor on {index.device}; got "
                         f"{tuple(table.shape)} {table.dtype} on {table.device}")
    if not 1 <= table.shape[1] <= _lib.PAIR_MAX_WIDTH:
        raise ValueError(f"the width D must be in [1, {_lib.PAIR_MAX_WIDTH}]; got {table.shape[1]}")
    if index.numel() >= 1 << 31:
        raise ValueError(f"at most 2^31 - 1 tokens in one call; got {index.numel()}")
    if base is not None:
        if tuple(base.shape) != (*index.shape, table.shape[1]) or base.device != index.device:
            raise ValueError(f"base must be {(*index.shape, table.shape[1])} on {index.device}; got {tuple(base.shape)} on {base.device}")
        if dtype is not None and dtype is not base.dtype:
            raise ValueError(f"the result has base's type {base.dtype}; got dtype={dtype}")
        dtype = base.dtype
    dtype = dtype or table.dtype
    if dtype not in PK.DTYPES:
        raise ValueError(f"the embedding's type must be bfloat16, float16 or float32; got {dtype}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite; got {scale}")
    index = index.contiguous()
    if _needs_grad(table, base):
        if wrap is not None:
            raise ValueError(_NO_DTENSOR_GRADIENT)
        return _PairEmbedding.apply(index, table, base, float(scale), dtype)
    out = _run_embed(index, table, base, float(scale), dtype)
    return out if wrap is None else wrap(out)
