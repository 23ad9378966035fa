"""Oracle of the pair-stream operators in 64 bits -- TEST INFRASTRUCTURE, not a compute path.

Restates, from the formulas and on whatever device its inputs live: the dropout's mask (Philox4x32-10 in numpy, pinned to
the published known answers by the tests), the residual's addition, the root-mean-square norm and its gradients, the e4m3
scaling, and the embedding with its gradient.  The norm takes the stored stream, as the operators do."""
from __future__ import annotations

import numpy as np
import torch

_M0, _M1, _W0, _W1 = (np.uint64(v) for v in (0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85))
_LOW = np.uint64(0xFFFFFFFF)
_32 = np.uint64(32)


def philox4x32_10(counter, key):
    """Four output words of four counter words (arrays of uint64 below 2^32) and two key words."""
    c = [np.asarray(w, dtype=np.uint64) for w in counter]
    k = [np.uint64(w) for w in key]
    for _ in range(10):
        p0, p1 = c[0] * _M0, c[2] * _M1
        c = [(p1 >> _32) ^ c[1] ^ k[0], p1 & _LOW, (p0 >> _32) ^ c[3] ^ k[1], p0 & _LOW]
        k = [(k[0] + _W0) & _LOW, (k[1] + _W1) & _LOW]
    return c


def keep_mask(shape, p, seed, offset=0, shared=None, origin=(0, 0, 0)):
    """``(bool mask, gain)`` of a ``(B, N_i, N_j, D)`` block that begins at ``origin`` of the grid."""
    B, I, J, D = shape
    b, i, j, v = np.ix_(*(np.arange(n, dtype=np.uint64) + np.uint64(o) for n, o in zip((B, I, J, (D + 7) // 8), (*origin, 0))))
    if shared == "rows":
        i = i * np.uint64(0)
    if shared == "columns":
        j = j * np.uint64(0)
    words = philox4x32_10([(b << np.uint64(16)) | v, j, i, np.uint64(offset)], [seed & 0xFFFFFFFF, seed >> 32])
    words = np.stack(np.broadcast_arrays(*words), axis=-1)
    halves = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], axis=-1)
    halves = np.broadcast_to(halves.reshape(*halves.shape[:3], -1)[..., :D], shape)
    keep = int(np.floor((1.0 - p) * 65536.0 + 0.5))
    return torch.from_numpy(halves < np.uint64(keep)), (65536.0 / keep if keep else 0.0)


def dropped(x, mask, gain):
    return torch.where(mask.to(x.device), x.double() * gain, torch.zeros((), dtype=torch.float64, device=x.device))


def rms_norm(z, weight, eps):
    z = z.double()
    return z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps) * weight.double()


def rms_norm_grad(z, weight, eps, dy, dz):
    """Gradients of the stream and of the gain, and the sums of absolute values that bound their rounding errors."""
    z, w, dy, dz = (t.double() for t in (z, weight, dy, dz))
    s = 1.0 / torch.sqrt(z.square().mean(-1, keepdim=True) + eps)
    t = w * dy
    g = dz + s * t - z * s ** 3 * (t * z).mean(-1, keepdim=True)
    g_abs = dz.abs() + (s * t).abs() + z.abs() * s ** 3 * (t * z).abs().mean(-1, keepdim=True)
    per_row = (dy * z * s).reshape(-1, z.shape[-1])
    return g, g_abs, per_row.sum(0), per_row.abs().sum(0)


def embedding(index, table, base, scale):
    index = index.long()
    there = (index >= 0) & (index < table.shape[0])
    rows = table.double()[index.where(there, torch.zeros_like(index))] * scale
    out = torch.where(there[..., None], rows, torch.zeros((), dtype=torch.float64, device=rows.device))
    return out if base is None else out + base.double()


def embedding_grad(index, rows, d_out, scale):
    """The table's gradient, and the sums of absolute values that bound its rounding error."""
    flat, d = index.reshape(-1).long(), d_out.reshape(-1, d_out.shape[-1]).double()
    there = (flat >= 0) & (flat < rows)
    sums = torch.zeros((2, rows, d.shape[1]), dtype=torch.float64, device=d.device)
    sums[0].index_add_(0, flat[there], d[there])
    sums[1].index_add_(0, flat[there], d[there].abs())
    return sums[0] * scale, sums[1] * abs(scale)
