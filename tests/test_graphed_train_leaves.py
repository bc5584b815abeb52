"""GraphedTrain refuses leaves whose earlier autograd graph is alive: captured into a graph, its backward pass ends the process.
Only the refusal and calls without such a graph run."""
import types

import pytest
import torch

from cagnet_amd import gcn


def test_live_graphs_of_a_leaf_are_found():
    w = torch.ones(3, requires_grad=True)
    assert not gcn._recorded_elsewhere(w) and not gcn._recorded_elsewhere(w)
    y = (w * 2).sum()
    assert gcn._recorded_elsewhere(w) and gcn._recorded_elsewhere(w)
    y.backward()
    kept = y.detach()
    assert gcn._recorded_elsewhere(w)  # the node outlives the buffers that backward freed
    del y
    assert not gcn._recorded_elsewhere(w) and kept.item() == 6.0
    w.grad = None
    assert not gcn._recorded_elsewhere(torch.ones(3)) and not gcn._recorded_elsewhere(w * 2)


@pytest.mark.parametrize("which", ["inputs", "weight1", "weight2"])
def test_refused_before_anything_runs(which):
    leaves = {k: torch.ones(4, 4, requires_grad=True) for k in ("inputs", "weight1", "weight2")}
    out = leaves[which] * 2  # noqa: F841
    with pytest.raises(RuntimeError, match=f"{which}: outputs computed from it earlier"):
        gcn.GraphedTrain(*leaves.values(), 4, [], None, None)


@pytest.mark.gpu
def test_eager_epochs_before_a_captured_one(cuda):
    from cagnet_amd import ops, synth

    p = synth.make_problem(scale=8, n_edges=1500, features=20, hidden=16, classes=6, mask_fraction=0.6, seed=2)
    blk = ops.CsrMatrix(p.row.int().to(cuda), p.col.int().to(cuda), p.val.to(cuda), p.n, p.n, transpose=True)
    data = types.SimpleNamespace(y=p.y.to(cuda), train_mask=p.train_mask.to(cuda))

    def fresh():
        w1, w2 = (w.to(cuda).requires_grad_() for w in (p.w1, p.w2))
        return p.x.to(cuda).requires_grad_(), w1, w2, torch.optim.SGD([w1, w2], lr=0.05), gcn.rng_state(4, cuda)

    x, w1, w2, opt, state = fresh()
    for _ in range(6):
        last = gcn.train(x, w1, w2, p.n, [blk], opt, data, dropout_p=0.4, rng=state).detach()
        x.grad = None
    x, g1, g2, opt, state = fresh()
    out = gcn.train(x, g1, g2, p.n, [blk], opt, data, dropout_p=0.4, rng=state)
    assert out.grad_fn is None  # with the loss fused into the last layer the outputs hold no graph and may be kept
    hidden = g1.square().sum()
    assert gcn._recorded_elsewhere(g1)
    with pytest.raises(RuntimeError, match="weight1: outputs computed from it earlier"):
        gcn.GraphedTrain(x, g1, g2, p.n, [blk], opt, data, dropout_p=0.4, rng=state)
    assert state.tolist() == [4, 1]
    del hidden
    x.grad = None
    graphed = gcn.GraphedTrain(x, g1, g2, p.n, [blk], opt, data, warmup=2, dropout_p=0.4, rng=state)
    for _ in range(3):
        got = graphed.step()
        torch.cuda.synchronize()
    assert torch.allclose(got, last, atol=1e-5) and torch.allclose(g1, w1, atol=1e-5) and torch.allclose(g2, w2, atol=1e-5)
    assert state.tolist() == [4, 6]
    graphed.close()
