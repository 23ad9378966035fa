"""The pair-stream operators on DTensors, host side: four gloo ranks on a 2 x 2 grid (and on a row split with a ragged last
block), with a stand-in for the native host module that draws the mask from the oracle at the position it is handed.  What the
ranks assemble has to be what one process draws for the whole grid."""
import os
import struct
import sys
import time
import traceback
from pathlib import Path

import pytest
import torch
import torch.multiprocessing as mp

REPO = Path(__file__).resolve().parent.parent


class _OracleHost:
    """Stands in for `_pair_host`: the same calls on CPU tensors, from the oracle."""

    def dropout_add(self, update, residual, drop, seed, out):
        from oracle.pair_oracle import dropped, keep_mask

        z = update.double()
        if drop:
            value, offset, keep, _, shared, *origin = struct.unpack("@QIIP4i", drop)
            mask, gain = keep_mask(tuple(update.shape), 1 - keep / 65536, value, offset, (None, "rows", "columns")[shared], origin)
            z = dropped(update, mask, gain)
        return (z if residual is None else z + residual.double()).to(update.dtype)

    def add_rms_norm(self, update, residual, weight, eps, drop, seed):
        from oracle.pair_oracle import rms_norm

        z = self.dropout_add(update, residual, drop, seed, None)
        return rms_norm(z, weight, eps).to(z.dtype), z

    def add_rms_norm_fp8(self, update, residual, weight, eps, group, drop, seed):
        y, z = self.add_rms_norm(update, residual, weight, eps, drop, seed)
        scales = y.abs().unflatten(-1, (-1, group or y.shape[-1])).amax(-1) / 448
        return y, scales, z

    def pair_embedding(self, index, table, scale, base, dtype):
        from oracle.pair_oracle import embedding

        return embedding(index, table, base, scale).to(dtype or table.dtype)


def _ranks(rank, world):
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import DTensor, Partial, Replicate, Shard, distribute_tensor

    from fold_cp_ops_b200 import _lib
    from fold_cp_ops_b200.workflows import pair_stream as P

    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        host = _OracleHost()
        _lib.pair_host = lambda: host
        g = torch.Generator().manual_seed(5)
        x, r = (torch.randn(2, 12, 10, 32, generator=g) for _ in range(2))
        w, index, table = torch.randn(32, generator=g), torch.randint(-1, 7, (2, 12, 10), generator=g), torch.randn(7, 32, generator=g)
        meshes = [(init_device_mesh("cpu", (2, 2)), (Shard(1), Shard(2))), (init_device_mesh("cpu", (4,)), (Shard(2),)),
                  (init_device_mesh("cpu", (2, 2)), (Shard(0), Shard(1))), (init_device_mesh("cpu", (4,)), (Replicate(),))]
        for mesh, placements in meshes:
            dx, dr = (distribute_tensor(t, mesh, placements) for t in (x, r))
            di = distribute_tensor(index, mesh, placements)
            at = P.pair_block_origin(dx)
            n = dx.to_local().shape
            assert torch.equal(dx.to_local(), x[at[0]:at[0] + n[0], at[1]:at[1] + n[1], at[2]:at[2] + n[2]])
            for shared in (None, "rows", "columns"):
                drop = P.PairDropout(0.25, seed=99, offset=4, shared=shared)
                want = host.dropout_add(x, r, P._record(drop, None)[0], None, None)
                z = P.dropout_add(dx, dr, drop)
                assert isinstance(z, DTensor) and z.placements == placements and torch.equal(z.full_tensor(), want)
                y, z = P.add_rms_norm(dx, dr, w, dropout=drop)
                assert torch.equal(z.full_tensor(), want) and y.shape == x.shape
                q, scales, z = P.add_rms_norm_fp8(dx, dr, w, group=32, dropout=drop)
                assert q.full_tensor().shape == x.shape and scales.full_tensor().shape == (2, 12, 10, 1)
            assert torch.equal(P.pair_embedding(di, table, base=dx).full_tensor(), host.pair_embedding(index, table, 1.0, x, None))
            whole = distribute_tensor(w, mesh, [Replicate()] * mesh.ndim)
            assert torch.equal(P.add_rms_norm(dx, None, whole)[0].full_tensor(), P.add_rms_norm(dx, None, w)[0].full_tensor())
        mesh, placements = meshes[0]
        dx = distribute_tensor(x, mesh, placements)
        bad = [lambda: P.dropout_add(dx, r), lambda: P.dropout_add(dx, distribute_tensor(r, mesh, (Shard(2), Shard(1)))),
               lambda: P.dropout_add(distribute_tensor(x, mesh, (Shard(1), Shard(3)))),
               lambda: P.dropout_add(DTensor.from_local(x, mesh, (Replicate(), Partial()))),
               lambda: P.dropout_add(distribute_tensor(x[0], mesh, (Shard(0), Shard(1)))),
               lambda: P.dropout_add(dx.detach().requires_grad_()), lambda: P.add_rms_norm(dx, None, w.clone().requires_grad_()),
               lambda: P.pair_embedding(distribute_tensor(index, mesh, placements), table.clone().requires_grad_()),
               lambda: P.add_rms_norm(dx, None, distribute_tensor(w, mesh, (Shard(0), Replicate()))),
               lambda: P.add_rms_norm(dx, None, distribute_tensor(w, mesh, (Replicate(), Replicate())).requires_grad_())]
        for k, call in enumerate(bad):
            try:
                call()
            except ValueError:
                continue
            raise AssertionError(f"call {k} was not refused")
        return "ok"
    finally:
        dist.destroy_process_group()


def _worker(rank, world, port, q):
    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world), MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    if str(REPO) not in sys.path:
        sys.path.insert(0, str(REPO))
    try:
        q.put((rank, _ranks(rank, world)))
    except BaseException as exc:  # noqa: BLE001 - reported to the parent
        q.put((rank, f"{type(exc).__name__}: {exc}\n{traceback.format_exc()}"))


def test_dtensors_on_four_ranks():
    import socket

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, 4, port, q)) for r in range(4)]
    for p in procs:
        p.start()
    out, deadline = {}, time.time() + 120
    while len(out) < 4 and time.time() < deadline:
        try:
            rank, res = q.get(timeout=1.0)
            out[rank] = res
        except Exception:
            if not any(p.is_alive() for p in procs) and q.empty():
                break
    for p in procs:
        p.join(timeout=10)
        if p.is_alive():
            p.terminate()
    assert out == {r: "ok" for r in range(4)}, out
