"""DTensors whose local block is still on its way: the host module gets the block itself, not the handle that stands for it."""
import os
import sys
import traceback
from pathlib import Path

import torch
import torch.multiprocessing as mp

REPO = Path(__file__).resolve().parent.parent


def _rank(rank, world, store):
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import Replicate, Shard, distribute_tensor

    from fold_cp_ops_b200 import _lib
    from fold_cp_ops_b200.workflows import pair_stream as P

    class Host:
        """Takes what the library can take: tensors with memory."""

        def add_rms_norm(self, update, residual, weight, eps, drop, seed):
            assert all(type(t) is torch.Tensor and t.data_ptr() != 0 for t in (update, residual, weight)), [type(t) for t in (update, residual, weight)]
            return update + 1, update + residual

    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=world)
    try:
        host = Host()
        _lib.pair_host = lambda: host
        mesh = init_device_mesh("cpu", (world,))
        x, w = torch.arange(2.0 * 4 * 4 * 8).reshape(2, 4, 4, 8), torch.arange(8.0)
        with torch.no_grad():
            rows = distribute_tensor(x, mesh, (Shard(1),))
            late = rows.redistribute(placements=(Shard(2),), async_op=True)
            gain = distribute_tensor(w, mesh, (Shard(0),)).redistribute(placements=(Replicate(),), async_op=True)
            y, z = P.add_rms_norm(late, distribute_tensor(x, mesh, (Shard(2),)), gain)
            assert torch.equal(y.full_tensor(), x + 1) and torch.equal(z.full_tensor(), 2 * x)
        return "ok"
    finally:
        dist.destroy_process_group()


def _worker(rank, world, store, q):
    if str(REPO) not in sys.path:
        sys.path.insert(0, str(REPO))
    os.environ.setdefault("GLOO_SOCKET_IFNAME", "lo")
    try:
        q.put((rank, _rank(rank, world, store)))
    except BaseException as exc:  # noqa: BLE001 - reported to the parent
        q.put((rank, f"{type(exc).__name__}: {exc}\n{traceback.format_exc()}"))


def test_blocks_that_are_still_on_their_way(tmp_path):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, 2, str(tmp_path / "store"), q)) for r in range(2)]
    for p in procs:
        p.start()
    out = dict(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(timeout=10)
        if p.is_alive():
            p.terminate()
    assert out == {0: "ok", 1: "ok"}, out
