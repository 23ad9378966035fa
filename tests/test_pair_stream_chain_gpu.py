"""The sort of the table's gradient in three and four digits: its buffers are rewritten within a call and reused by the next."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("rows", [70000, (1 << 24) + 3])
@pytest.mark.parametrize("n", [20011, 300007])
def test_gradients_of_large_tables_one_behind_another(rows, n):
    """Whole numbers below 2^24 / n add up without rounding: every call has to give the sums exactly."""
    from fold_cp_ops_b200.workflows import pair_stream as p

    table = torch.zeros(rows, 2, device=DEV, requires_grad=True)
    got, want = [], []
    for k in range(8):
        g = torch.Generator(device=DEV).manual_seed(k)
        index = (torch.rand(n, generator=g, device=DEV) ** (1, 6)[k % 2] * rows).long().clamp(0, rows - 1)
        index[k::7] = -1
        d_out = torch.randint(-20, 21, (n, 2), generator=g, device=DEV).float()
        got.append(torch.autograd.grad(p.pair_embedding(index, table), table, d_out)[0].long().to_sparse())
        there = index >= 0
        want.append(torch.zeros(rows, 2, dtype=torch.int64, device=DEV).index_add_(0, index[there], d_out[there].long()).to_sparse())
    for k, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a.to_dense(), b.to_dense()), f"call {k}"
