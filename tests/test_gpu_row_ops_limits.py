"""Calls of the row-wise training operators at the ends of what they take."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _memory_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("cols", [(1 << 31), (1 << 32) + 16])
def test_rows_of_more_columns_than_the_abi_counts(cuda, cols):
    """Refused before anything is copied or allocated: 2^32 + 16 columns would arrive as 16."""
    from cagnet_amd import gcn, ops

    x = torch.ones(1, 1, device=cuda).expand(1, cols)
    idx, rstd = torch.zeros(1, dtype=torch.int64, device=cuda), torch.ones(1, device=cuda)
    for call in (lambda: ops.dropout_fwd(x, 0.0, None), lambda: ops.embedding_fwd(x, idx), lambda: ops.embedding_bwd(x, idx, 1),
                 lambda: ops.rms_norm_fwd(x, None), lambda: ops.rms_norm_bwd(x, x, None, rstd),
                 lambda: ops.norm_residual_fwd(x, x, None, None), lambda: gcn.rms_norm(x, None)):
        with pytest.raises(ValueError, match="at most 2147483647"):
            call()


def test_embedding_of_the_most_indices(cuda):
    """2^31 - 2^20 - 1 indices of five rows.  The gradient is zero but at 4,000 positions and both ends, so that its sums are
    exact in any order."""
    from cagnet_amd import ops

    n = (1 << 31) - (1 << 20) - 1
    gen = torch.Generator(device=cuda).manual_seed(1)
    idx = torch.randint(-1, 6, (n,), dtype=torch.int32, device=cuda, generator=gen)
    table = torch.tensor([[1.0], [2.0], [3.0], [4.0], [5.0]], dtype=torch.bfloat16, device=cuda)
    out = ops.embedding_fwd(table, idx)
    lookup = torch.tensor([0, 1, 2, 3, 4, 5, 0], dtype=torch.bfloat16, device=cuda)
    for at in (0, n // 2, n - 5_000_000):
        part = slice(at, at + 5_000_000)
        assert torch.equal(out[part, 0], lookup[idx[part].long() + 1])
    g = out.zero_()
    marked = torch.cat([torch.randperm(100_000_000, device=cuda, generator=gen)[:4000] * 21, torch.tensor([1, 2, 3, n - 2, n - 1], device=cuda)])
    marked = marked[marked < n].unique()
    g[marked, 0] = 1.0
    got = ops.embedding_bwd(g, idx, 5, out=torch.empty(5, 1, device=cuda))
    named = idx[marked].long()
    want = torch.bincount(named[(named >= 0) & (named < 5)], minlength=5)
    assert got[:, 0].tolist() == want.tolist()


def test_embedding_gradient_of_a_large_table(cuda):
    """40 million indices into 9 million rows: three passes of the sort over many tiles, whole numbers."""
    from cagnet_amd import ops

    n, rows = 40_000_000, 9_000_000
    gen = torch.Generator(device=cuda).manual_seed(2)
    idx = (torch.rand(n, device=cuda, generator=gen) ** 4 * (rows + 1)).int()
    idx[:1_000_000] = 77
    g = torch.randint(1, 9, (n, 2), device=cuda, generator=gen).float()
    want = torch.zeros(rows + 2, 2, dtype=torch.int64, device=cuda).index_add_(0, idx.long(), g.long())[:rows]
    assert int(want.max()) < 1 << 24
    for beta in (0.0, 1.0):
        out = torch.ones(rows, 2, device=cuda)
        ops.embedding_bwd(g, idx, rows, out=out, beta=beta)
        assert torch.equal(out.long(), want + int(beta))


def test_most_rows(cuda):
    """2^32 - 1 rows of one element: the generator's row counter is used to its end."""
    from cagnet_amd import ops
    from oracle import row_ops_oracle as ref

    n = (1 << 32) - 1
    x = torch.ones(n, 1, dtype=torch.bfloat16, device=cuda)
    got = ops.dropout_fwd(x, 0.25, ops.rng_state(6, cuda, 2))
    for row0 in (0, (1 << 31) - 3, n - 7):
        assert torch.equal(got[row0:row0 + 7].cpu().float() != 0, ref.keep_mask(6, 2, 7, 1, 0.25, row0=row0)), row0
    del got
    x[-1] = 0.0
    y, rstd = ops.rms_norm_fwd(x, None)
    assert bool((y[:-1] == 1).all()) and float(y[-1]) == 0.0 and abs(float(rstd[-1]) - 1000.0) < 1e-3
    with pytest.raises(ops.CagnetError, match="CG_ERR_OVERFLOW"):
        ops.dropout_fwd(torch.empty(n + 1, 1, dtype=torch.bfloat16, device=cuda), 0.0, None)


def test_longest_rows(cuda):
    """2^31 - 1 columns of dropout, 2^30 of the norms, 2^23 of the embedding."""
    import numpy as np

    from cagnet_amd import ops
    from oracle import row_ops_oracle as ref

    d = (1 << 31) - 1
    got = ops.dropout_fwd(torch.ones(1, d, dtype=torch.bfloat16, device=cuda), 0.25, ops.rng_state(6, cuda, 2))
    for block in (0, (1 << 28) + 5, (d - 1) // 4):
        words = ref.philox([np.uint64(block), np.uint64(0), np.uint64(2), np.uint64(0)], [6, 0])
        live = min(4, d - 4 * block)
        want = [int(w) >= 1 << 30 for w in words][:live]
        assert (got[0, 4 * block:4 * block + live] != 0).tolist() == want, block
    del got
    d = 1 << 30
    x = torch.ones(1, d, dtype=torch.bfloat16, device=cuda)
    y, rstd = ops.rms_norm_fwd(x, None)
    assert bool((y == 1).all()) and abs(float(rstd[0]) - 1) < 1e-5
    dx, dw = ops.rms_norm_bwd(x, x, y[0], rstd)
    assert float(dx.abs().max()) < 1e-4 and bool((dw == 1).all())
    del y, dx, dw
    w = torch.full((d,), 2.0, dtype=torch.bfloat16, device=cuda)
    r, h, rstd_z, rstd_r = ops.norm_residual_fwd(x, x, w, None)
    assert bool((r == 3).all()) and bool((h == 1).all()) and abs(float(rstd_r[0]) - 1 / 3) < 1e-5
    dz, dx, _, dw, _, _ = ops.norm_residual_bwd(x, None, x, r, w, None, rstd_z, rstd_r)
    assert float(dz.abs().max()) < 1e-4 and torch.equal(dx, x) and bool((dw == 1).all())
    del x, w, r, h, dz, dx, dw
    d = 1 << 23
    table = torch.arange(3 * d, device=cuda).reshape(3, d) % 64
    idx = torch.tensor([2, 0, 2, 3, 2] * 5, device=cuda)
    out = ops.embedding_fwd(table.bfloat16(), idx)
    assert torch.equal(out[0], table[2].bfloat16()) and torch.equal(out[1], table[0].bfloat16()) and not bool(out[3].any())
    grad = ops.embedding_bwd(out, idx, 3, out=torch.empty(3, d, device=cuda))
    assert torch.equal(grad, table * torch.tensor([[5.0], [0.0], [15.0]], device=cuda))
