"""Calls of the row-wise training operators at the ends of what they take."""
import pytest
import torch

pytestmark = pytest.mark.gpu


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
