"""The pair stream around the triangle update: what makes it, what is added to it, what reads it.

A pair stack keeps one representation ``z`` of shape ``(B, N_i, N_j, D)``.  The triangle update (this package's other
operators) computes an update of it; the functions here are the rest of the stream, each one pass over HBM:

* :func:`dropout_add` -- ``z = residual + dropout(update)``;
* :func:`add_rms_norm` -- the same, and the root-mean-square norm of ``z`` that the next block reads;
* :func:`add_rms_norm_fp8` -- the same with the norm in e4m3 and fp32 scales, for an 8-bit product;
* :func:`pair_embedding` -- ``base + scale * table[index]``: position or distance bins, residue types.

All but the e4m3 form have gradients (once; backwards only: inputs with forward-mode tangents, and calls under a tracer, are refused).  Statistics and sums are fp32 or wider whatever the tensors'
type, and there values below 2^-126 count as 0; ``z`` is rounded once, to the activations' type and its subnormals, and the norm reads ``z`` as it is stored.

Dropout (:class:`PairDropout`) stores no mask: element ``(b, i, j, c)`` of the WHOLE grid is kept by a counter-based
generator of exactly that position, so the gradient draws the mask again, and ranks that hold different blocks of a
context-parallel grid draw the same mask as one GPU would.

Tensors may be DTensors sharded over batch and token dims, as the distributed triangle update takes them: the blocks'
positions are then taken from the placements, and gains and tables may be replicated DTensors.  Gradients are for plain
tensors only; those of gains and tables are of the block that was passed, to be added up over ranks.  Inputs need contiguous channels
(others are copied); other strides -- a transposed view, a block of a larger tensor, a broadcast axis -- are read in place.
There is no CPU path.
"""
from __future__ import annotations

import math
import operator
import struct
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from .. import _lib
from ..distributed.dtensor_adapter import (_dtensor_mesh_placements, _effective_placements, _is_dtensor, _rowmaj_stride,
                                           _shards)

__all__ = ["PairDropout", "dropout_add", "add_rms_norm", "add_rms_norm_fp8", "pair_embedding", "pair_block_origin"]

_SHARED = {None: 0, "rows": 1, "columns": 2}
_PLAIN = frozenset((Tensor, torch.nn.Parameter, type(None)))
_NO_DTENSOR_GRADIENT = "gradients through DTensors are not supported: pass the local blocks, with PairDropout.origin"

#: a ``pair_dropout_t`` of include/pair_stream_sm100.h: seed, offset, keep, (device seed), shared, origin b, i, j
_pack_dropout = struct.Struct("@QIIP4i").pack
_NO_DROPOUT = (b"", None)


def _fits(value, bits: int) -> bool:
    try:
        return 0 <= operator.index(value) < 1 << bits
    except TypeError:
        return False


@dataclass(frozen=True)
class PairDropout:
    """A dropout of pair tensors whose mask is a function of its arguments alone.

    ``p``: probability of being dropped, in multiples of 2^-16 (the nearest is taken); kept elements are multiplied by the
    exact reciprocal of the probability of being kept.  ``seed`` (64 bits) and ``offset`` (32 bits) name the mask: give every
    layer and step its own pair.  For captured graphs ``seed`` may be a CUDA tensor of two int64 values ``[seed, offset]``
    that is read when the kernel runs (``offset`` is then ignored here); it must keep its values until the gradient is computed.
    ``shared``: ``"rows"`` -- one mask for all rows ``i``; ``"columns"`` -- one for all columns ``j``; ``None`` -- every
    element its own.  ``origin``: the ``(b, i, j)`` of the tensor's first element in the whole grid, where the tensor is one
    rank's block (DTensors know theirs).  At most 65536 batch entries."""

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
        elif not _fits(self.seed, 64):
            raise ValueError(f"seed must be an integer of 64 bits, unsigned; got {self.seed!r}")
        if not _fits(self.offset, 32):
            raise ValueError(f"offset must be an integer of 32 bits, unsigned; got {self.offset!r}")
        if len(self.origin) != 3 or not all(_fits(o, 31) for o in self.origin):
            raise ValueError(f"origin must be three integers (b, i, j), >= 0 and below 2^31; got {self.origin!r}")

    @property
    def keep(self) -> int:
        """How many of 65536 values are kept."""
        return math.floor((1.0 - self.p) * 65536.0 + 0.5)


def _record(dropout: Optional[PairDropout], wrap: Optional["_Wrap"]) -> Tuple[bytes, Optional[Tensor]]:
    """The library's record of a dropout (empty where everything is kept), at the position of this rank's block, and the
    device seed."""
    if dropout is None:
        return _NO_DROPOUT
    if not isinstance(dropout, PairDropout):
        raise TypeError(f"dropout must be a PairDropout or None; got {type(dropout).__name__}")
    keep = dropout.keep
    if keep == 65536:
        return _NO_DROPOUT
    origin = dropout.origin
    if wrap is not None:
        origin = tuple(o + at for o, at in zip(origin, pair_block_origin(wrap.like)))
        if not all(_fits(o, 31) for o in origin):
            raise ValueError(f"the dropout's origin {dropout.origin} puts this block at {origin}, behind 2^31 - 1")
    seed, offset, device_seed = dropout.seed, dropout.offset, None
    if isinstance(seed, Tensor):
        seed, offset, device_seed = 0, 0, seed
    return _pack_dropout(seed, offset, keep, 0, _SHARED[dropout.shared], *origin), device_seed


def pair_block_origin(x) -> Tuple[int, int, int]:
    """``(b, i, j)`` of this rank's first element of a pair DTensor in the whole grid."""
    from torch.distributed.tensor._utils import compute_local_shape_and_global_offset

    mesh, placements = _dtensor_mesh_placements(x)
    _, offset = compute_local_shape_and_global_offset(x.shape, mesh, placements)
    return tuple(int(o) for o in offset[:3])


# ---------------------------------------------------------------------------------------------
# DTensors
# ---------------------------------------------------------------------------------------------
def _local(t) -> Tensor:
    """This rank's block, waited for where the collective that makes it is still under way."""
    local = t.to_local()
    return local.trigger_wait() if hasattr(local, "trigger_wait") else local


def _locals_of(names: Sequence[str], tensors: Sequence[Optional[Tensor]]):
    """The ranks' local blocks of DTensors that are sharded alike, and their :class:`_Wrap` (``None`` where all are plain)."""
    given = [(n, t) for n, t in zip(names, tensors) if t is not None]
    if not any(_is_dtensor(t) for _, t in given):
        return tensors, None
    if not all(_is_dtensor(t) for _, t in given):
        raise ValueError(f"{', '.join(n for n, _ in given)} must be DTensors of the same placements or all plain tensors")
    if torch.is_grad_enabled() and any(t.requires_grad for _, t in given):
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
    return [None if t is None else _local(t) for t in tensors], _Wrap(mesh, placements, x, tokens)


class _Wrap:
    """Makes local results DTensors again."""

    def __init__(self, mesh, placements, like, tokens: int):
        self.mesh, self.placements, self.like, self.tokens = mesh, placements, like, tuple(like.shape[:tokens])

    def __call__(self, local: Tensor):
        from torch.distributed.tensor import DTensor

        shape = torch.Size((*self.tokens, *local.shape[len(self.tokens):]))
        return DTensor.from_local(local, self.mesh, self.placements, run_check=False, shape=shape, stride=_rowmaj_stride(shape))


def _whole(t, name: str):
    """A parameter that may be a replicated DTensor, as this rank holds it."""
    if type(t) in _PLAIN or not _is_dtensor(t):
        return t
    if any(not p.is_replicate() for p in _effective_placements(*_dtensor_mesh_placements(t))):
        raise ValueError(f"{name} must be whole on every rank; got placements {_dtensor_mesh_placements(t)[1]}")
    if torch.is_grad_enabled() and t.requires_grad:
        raise ValueError(_NO_DTENSOR_GRADIENT)
    return _local(t)


def _no_gradient(wrap: Optional[_Wrap], *parameters: Tensor) -> None:
    if wrap is not None and torch.is_grad_enabled() and any(t.requires_grad for t in parameters):
        raise ValueError(_NO_DTENSOR_GRADIENT)


# ---------------------------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------------------------
def dropout_add(update: Tensor, residual: Optional[Tensor] = None, dropout: Optional[PairDropout] = None, *,
                out: Optional[Tensor] = None) -> Tensor:
    """``residual + dropout(update)`` in the tensors' type (bfloat16, float16 or float32), rounded once.

    ``update`` and ``residual``: ``(B, N_i, N_j, D)`` or its last dims, of one shape, type and device, any strides, ``D`` at
    most 8192.  ``residual=None`` is a plain dropout.  ``out`` (contiguous; no gradients) may be ``residual`` or ``update``
    itself: the stream is then updated in place.  Dropped elements become 0 whatever they were.  Raises ``ValueError`` for
    anything else, ``TypeError`` for a ``dropout`` that is no :class:`PairDropout`."""
    given, wrap = out, None
    if type(update) not in _PLAIN or type(residual) not in _PLAIN or type(out) not in _PLAIN:
        (update, residual, out), wrap = _locals_of(("update", "residual", "out"), (update, residual, out))
    drop, seed = _record(dropout, wrap)
    z = _lib.pair_host().dropout_add(update, residual, drop, seed, out)
    if given is not None:
        return given
    return z if wrap is None else wrap(z)


def add_rms_norm(update: Tensor, residual: Optional[Tensor], weight: Tensor, *, eps: float = 1e-5,
                 dropout: Optional[PairDropout] = None) -> Tuple[Tensor, Tensor]:
    """``(y, z)``: ``z = residual + dropout(update)`` and ``y = z / sqrt(mean(z^2) + eps) * weight`` over the channels.

    Tensors as in :func:`dropout_add`; ``weight`` is ``(D,)`` in any of the three types and gets its gradient in its own.
    ``residual=None`` takes the norm of ``dropout(update)``; without a dropout too, ``z`` is ``update`` itself."""
    wrap = None
    if type(update) not in _PLAIN or type(residual) not in _PLAIN:
        (update, residual), wrap = _locals_of(("update", "residual"), (update, residual))
        _no_gradient(wrap, weight)
    drop, seed = _record(dropout, wrap)
    y, z = _lib.pair_host().add_rms_norm(update, residual, _whole(weight, "weight"), eps, drop, seed)
    return (y, z) if wrap is None else (wrap(y), wrap(z))


def add_rms_norm_fp8(update: Tensor, residual: Optional[Tensor], weight: Tensor, *, eps: float = 1e-5,
                     group: Optional[int] = 128, dropout: Optional[PairDropout] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """``(q, scales, z)``: :func:`add_rms_norm` with ``y`` in ``float8_e4m3fn``, ``y ~ q * scales`` per ``group`` channels.

    ``group`` is 32, 64 or 128 (dividing ``D``), or ``None`` for one scale per row; ``scales`` is fp32,
    ``(..., D / group)``: the group's largest ``|y|`` / 448, at least 2^-126, and 1 for a group of zeros.  ``q`` is the quotient
    ``y / scale`` rounded once, ties to even: of 16-bit tensors with a 16-bit ``weight`` the exact quotient to within 2^-24 of it (a tie
    stays a tie), of others to within a few 2^-24.  For inference: refuses inputs that require gradients.  Scales per group need rows that start on 16-byte
    boundaries; other inputs are copied first."""
    wrap = None
    if type(update) not in _PLAIN or type(residual) not in _PLAIN:
        (update, residual), wrap = _locals_of(("update", "residual"), (update, residual))
    drop, seed = _record(dropout, wrap)
    q, scales, z = _lib.pair_host().add_rms_norm_fp8(update, residual, _whole(weight, "weight"), eps, group, drop, seed)
    return (q, scales, z) if wrap is None else (wrap(q), wrap(scales), wrap(z))


def pair_embedding(index: Tensor, table: Tensor, *, scale: float = 1.0, base: Optional[Tensor] = None,
                   dtype: Optional[torch.dtype] = None) -> Tensor:
    """``base + scale * table[index]``: an embedding lookup into the pair stream, ``(*index.shape, D)``.

    ``index``: int32 or int64, any shape; an entry outside ``[0, V)`` (``-1`` for padding) adds nothing and gets no gradient.
    ``table``: ``(V, D)`` in bfloat16, float16 or float32, ``D`` at most 8192; its gradient comes in its type, summed in at
    least fp32 and in a fixed order (the same bits every time).  ``base``: what the embedding is
    added to, or ``None``; the result has its type, else ``dtype``, else the table's.  ``index`` and ``base`` may be DTensors
    sharded alike.  ``index``, ``base`` and the result's gradient are copied where they are not contiguous."""
    wrap = None
    if type(index) not in _PLAIN or type(base) not in _PLAIN:
        (index, base), wrap = _locals_of(("index", "base"), (index, base))
        _no_gradient(wrap, table)
    out = _lib.pair_host().pair_embedding(index, _whole(table, "table"), scale, base, dtype)
    return out if wrap is None else wrap(out)
