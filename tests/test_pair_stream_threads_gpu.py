"""The C entries from two threads at once, each with its own stream, buffers and workspace."""
import ctypes as C
import threading

import pytest
import torch

from .test_pair_stream_cpu import EmbedDesc

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, FP32 = 0, 2


def test_gradients_of_small_tables_from_two_threads():
    """Tables of one and of 74 rows take 8 and 225 KB of shared memory of the same kernel.  Whole numbers: exact sums."""
    from fold_cp_ops_b200 import _lib

    lib, n, d, errors = _lib.load(), 8192, 64, []
    barrier = threading.Barrier(2)

    def work(rows):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            index = torch.arange(n, device=DEV) % rows
            d_out = torch.ones(n, d, device=DEV)
            out = torch.empty(rows, d, device=DEV)
            desc, size = EmbedDesc(n, d, rows, 64, FP32, FP32, 1.0), C.c_uint64()
            assert lib.pair_sm100_embed_grad_workspace(C.byref(desc), C.byref(size)) == 0
            workspace = torch.empty(size.value, dtype=torch.uint8, device=DEV)
            want = torch.bincount(index, minlength=rows)[:, None].expand(rows, d).float()
            stream.synchronize()
            barrier.wait()
            args = [C.byref(desc), *(C.c_void_p(t.data_ptr()) for t in (index, d_out, out, workspace)), C.c_void_p(stream.cuda_stream)]
            for k in range(20000):
                rc = lib.pair_sm100_embed_grad(*args)
                if rc != 0:
                    errors.append(f"{rows} rows, call {k}: code {rc}, {_lib.last_error()}")
                    break
            stream.synchronize()
            if not torch.equal(out, want):
                errors.append(f"{rows} rows: wrong sums")

    threads = [threading.Thread(target=work, args=(r,)) for r in (1, 74)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
