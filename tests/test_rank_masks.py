"""Ranks that share a seed drop different elements of their blocks in gcn.train."""
import types

import pytest
import torch

from oracle import row_ops_oracle as ref


def test_ranks_step_through_offsets_of_their_own():
    from cagnet_amd import gcn

    seen = set()
    for rank in (0, 1, 2, 7, 32767, 32768, 65535):
        snapshot = gcn._rank_masks(torch.tensor([-5, 9]), rank)
        seed, offset = snapshot.tolist()
        assert seed == -5 and offset % (1 << 64) == (rank << 48) + 9
        seen.add(offset)
    assert len(seen) == 7


@pytest.mark.gpu
def test_two_ranks_with_one_seed(cuda):
    """One epoch of each of two ranks of a 1D partition (the other's dense blocks resident) against 64 bits, masks of offset
    rank * 2^48; the ranks' masks differ where they kept the same ones before."""
    from cagnet_amd import gcn, ops, synth

    size, p_drop = 2, 0.5
    p = synth.make_problem(n=600, target_nnz=9000, features=20, hidden=16, classes=6, mask_fraction=0.6, seed=4)
    half = p.n // size
    A = torch.sparse_coo_tensor(torch.stack([p.row, p.col]), p.val.double(), (p.n, p.n)).to_dense()
    keeps = [ref.keep_mask(9, (r << 48) + 3, half, 16, p_drop) for r in range(size)]
    assert not torch.equal(*keeps)
    m1, m2 = p.w1.double(), p.w2.double()
    hidden = torch.relu(A @ p.x.double() @ m1)
    hidden = torch.where(torch.cat(keeps), hidden / (1 - p_drop), 0.0)
    want = torch.log_softmax(A @ hidden @ m2, 1)
    for r in range(size):
        rows = slice(r * half, (r + 1) * half)
        blocks = []
        for k in range(size):
            rr, cc, vv = synth.coo_block(p.row, p.col, p.val, r * half, (r + 1) * half, k * half, (k + 1) * half)
            blocks.append(ops.CsrMatrix(rr.int().to(cuda), cc.int().to(cuda), vv.to(cuda), half, half))
        mine = lambda t: [None if k == r else t[k * half:(k + 1) * half].float().to(cuda) for k in range(size)]  # noqa: E731
        zeros = lambda d: mine(torch.zeros(p.n, d))  # noqa: E731
        group = (gcn.ResidentBlocks(mine(p.x), zeros(16)), gcn.ResidentBlocks(mine(hidden), zeros(6)))
        w1, w2 = (w.to(cuda).requires_grad_() for w in (p.w1, p.w2))
        data = types.SimpleNamespace(y=p.y.to(cuda), train_mask=p.train_mask.to(cuda))
        state = gcn.rng_state(9, cuda, 3)
        out = gcn.train(p.x[rows].to(cuda).requires_grad_(), w1, w2, p.n, blocks, torch.optim.SGD([w1, w2], lr=0.0), data, r, size,
                        group, dropout_p=p_drop, rng=state)
        off = (out.detach().cpu().double() - want[rows]).abs().max()
        assert float(off) <= 2e-4 * float(want.abs().max()), (r, float(off))
        assert state.tolist() == [9, 4]


@pytest.mark.gpu
def test_masks_of_a_rank_in_a_captured_epoch(cuda):
    """Every replay steps the state once and takes the rank's next mask, with eager work in between."""
    from cagnet_amd import gcn

    state, x = gcn.rng_state(6, cuda, 40), torch.ones(50, 12, device=cuda)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = gcn.dropout(x, 0.4, gcn._rank_masks(gcn.rng_next(state), 3))
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu() != 0, ref.keep_mask(6, (3 << 48) + 40 + k, 50, 12, 0.4)), k
        assert float((x * 2).sum()) == 1200.0 and state.tolist() == [6, 41 + k]
