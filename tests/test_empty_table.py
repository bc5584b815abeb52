"""A lookup of no indices is legal whatever the table, an empty one included (a type of vertices that a graph does not have)."""
import ctypes

import pytest
import torch

SIZE = 2


def test_entry_points_take_no_indices_into_no_rows():
    from cagnet_amd._lib import lib

    size = ctypes.c_int64(-1)
    assert lib.cg_embedding_fwd(None, 8, 0, None, 1, 0, 8, 0, 1.0, None, 8, None) == 0
    assert lib.cg_embedding_bwd_workspace(0, 0, 8, ctypes.byref(size)) == 0 and size.value >= 0
    assert lib.cg_embedding_bwd(None, 8, None, 1, 0, 0, 8, 0, 0, 1.0, 0.0, None, 8, None, 0, None) == 0
    for n, rows, d in ((1, 0, 8), (0, -1, 8), (-1, 0, 8), (0, 0, 0)):  # an index has to have a table
        assert lib.cg_embedding_fwd(16, 8, rows, 16, 1, n, d, 0, 1.0, 4096, 8, None) == SIZE
        assert lib.cg_embedding_bwd_workspace(n, rows, d, ctypes.byref(size)) == SIZE
        assert lib.cg_embedding_bwd(16, 8, 16, 1, n, rows, d, 0, 0, 1.0, 0.0, 4096, 8, 4096, 1 << 20, None) == SIZE


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_empty_table_with_autograd(cuda, t):
    from cagnet_amd import gcn, ops

    table = torch.empty(0, 24, dtype=t, device=cuda, requires_grad=True)
    for shape in ((0,), (0, 3)):
        out = gcn.embedding(table, torch.empty(shape, dtype=torch.int64, device=cuda))
        assert out.shape == (*shape, 24)
        out.sum().backward()
        assert table.grad.shape == (0, 24)
    for beta in (0.0, 1.0, 0.5):
        out = torch.empty(0, 24, device=cuda)
        assert ops.embedding_bwd(table.detach(), torch.empty(0, dtype=torch.int32, device=cuda), 0, out=out, beta=beta) is out
