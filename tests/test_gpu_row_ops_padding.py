"""Outputs with leading dimensions larger than their rows, through the C ABI: the same bits as with rows side by side, and
nothing else written, in front of the first row, between rows and behind the last."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.bfloat16, torch.float16]
CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MARK = 77.0
SHAPES = [(9, 1), (11, 3), (300, 5), (37, 41), (300, 64), (23, 602), (9, 1027), (3, 2560), (3, 8201), (2, 16_384)]


class Padded:
    """An [n, d] output `front` elements into a buffer with rows `gap` elements apart."""

    def __init__(self, n, d, t, cuda, front=3, gap=5, fill=None):
        self.n, self.d, self.ld, self.front = n, d, d + gap, front
        self.buffer = torch.full((front + n * self.ld + 64,), MARK, dtype=t, device=cuda)
        self.window = self.buffer[front:front + n * self.ld].view(n, self.ld)[:, :d]
        if fill is not None:
            self.window.copy_(fill)

    def at(self):
        return self.window.data_ptr()

    def check(self, want, name):
        assert torch.equal(self.window, want), name
        self.window.fill_(MARK)
        assert bool((self.buffer == MARK).all()), f"{name}: written outside its rows"


def call(name, *args):
    from cagnet_amd._lib import lib

    assert getattr(lib, name)(*args, torch.cuda.current_stream().cuda_stream) == 0, name


def work(name, *sizes):
    from cagnet_amd._lib import lib

    need = ctypes.c_int64(0)
    assert getattr(lib, name)(*sizes, ctypes.byref(need)) == 0
    return torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("n,d", SHAPES)
def test_dropout(cuda, t, n, d):
    from cagnet_amd import ops

    x, rng = torch.randn(n, d, generator=torch.Generator().manual_seed(d)).to(t).to(cuda), ops.rng_state(5, cuda)
    for p in (0.0, 0.3):
        out = Padded(n, d, t, cuda)
        call("cg_dropout", x.data_ptr(), d, out.at(), out.ld, n, d, CODE[t], p, rng.data_ptr())
        out.check(ops.dropout_fwd(x, p, rng), f"p {p}")
        out = Padded(n, d, t, cuda, fill=x)  # in place
        call("cg_dropout", out.at(), out.ld, out.at(), out.ld, n, d, CODE[t], p, rng.data_ptr())
        out.check(ops.dropout_fwd(x, p, rng), f"in place, p {p}")


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("n,d", SHAPES)
def test_embedding(cuda, t, n, d):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(d)
    rows = 20
    table, g = torch.randn(rows, d, generator=gen).to(t).to(cuda), torch.randn(n, d, generator=gen).to(t).to(cuda)
    idx = torch.randint(-1, rows + 1, (n,), generator=gen).to(cuda)
    idx[n // 3:] = 7  # a hot row where there are indices enough
    out = Padded(n, d, t, cuda)
    call("cg_embedding_fwd", table.data_ptr(), d, rows, idx.data_ptr(), 1, n, d, CODE[t], 0.5, out.at(), out.ld)
    out.check(ops.embedding_fwd(table, idx, 0.5), "lookup")
    space = work("cg_embedding_bwd_workspace", n, rows, d)
    for ot in {t, torch.float32}:
        old = torch.randn(rows, d, generator=gen).to(ot).to(cuda)
        for beta in (0.0, 1.0, 0.25):
            out = Padded(rows, d, ot, cuda, fill=old)
            call("cg_embedding_bwd", g.data_ptr(), d, idx.data_ptr(), 1, n, rows, d, CODE[t], CODE[ot], 0.5, beta, out.at(), out.ld,
                 space.data_ptr(), space.numel())
            out.check(ops.embedding_bwd(g, idx, rows, 0.5, out=old.clone(), beta=beta), f"gradient {ot} {beta}")


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("d", [3, 30, 64, 130])
def test_embedding_gradient_of_many_indices(cuda, t, d):
    """The sort of several tiles, hot rows and rows that no index names."""
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(d)
    n, rows = 9000, 3000
    g, idx = torch.randn(n, d, generator=gen).to(t).to(cuda), torch.randint(-1, rows, (n,), generator=gen)
    idx[torch.rand(n, generator=gen) < 0.5] = 2
    idx = idx.to(cuda)
    space = work("cg_embedding_bwd_workspace", n, rows, d)
    old = torch.randn(rows, d, generator=gen).to(t).to(cuda)
    for beta in (0.0, 1.0, 0.25):
        out = Padded(rows, d, t, cuda, fill=old)
        call("cg_embedding_bwd", g.data_ptr(), d, idx.data_ptr(), 1, n, rows, d, CODE[t], CODE[t], 0.5, beta, out.at(), out.ld,
             space.data_ptr(), space.numel())
        out.check(ops.embedding_bwd(g, idx, rows, 0.5, out=old.clone(), beta=beta), f"{beta}")


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("n,d", SHAPES)
def test_rms_norm(cuda, t, n, d):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(d)
    x, g, w = (torch.randn(*s, generator=gen).to(t).to(cuda) for s in ((n, d), (n, d), (d,)))
    y, rstd, space = Padded(n, d, t, cuda), torch.full((n + 2,), MARK, device=cuda), work("cg_norm_bwd_workspace", n, d)
    call("cg_rms_norm_fwd", x.data_ptr(), d, w.data_ptr(), CODE[t], y.at(), y.ld, rstd[1:].data_ptr(), n, d, CODE[t], 1e-6)
    want_y, want_rstd = ops.rms_norm_fwd(x, w)
    y.check(want_y, "y")
    assert torch.equal(rstd[1:-1], want_rstd) and rstd[0] == MARK and rstd[-1] == MARK
    dx, dw = Padded(n, d, t, cuda), torch.full((d + 2,), MARK, dtype=t, device=cuda)
    call("cg_rms_norm_bwd", g.data_ptr(), d, x.data_ptr(), d, w.data_ptr(), CODE[t], want_rstd.data_ptr(), dx.at(), dx.ld,
         dw[1:].data_ptr(), n, d, CODE[t], space.data_ptr(), space.numel())
    want_dx, want_dw = ops.rms_norm_bwd(g, x, w, want_rstd)
    dx.check(want_dx, "dx")
    assert torch.equal(dw[1:-1], want_dw) and dw[0] == MARK and dw[-1] == MARK


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("n,d,kind", [(n, d, kind) for n, d in SHAPES for kind in (0, 1, 2) if kind < 2 or d > 1])  # [n, 1] is a row's
def test_norm_residual(cuda, t, n, d, kind):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(d)
    z, x, dr, dh = (torch.randn(n, d, generator=gen).to(t).to(cuda) for _ in range(4))
    w = [torch.randn(d, generator=gen).to(cuda) for _ in range(3)]
    width = (0, 1, d)[kind]
    gate = torch.randn(n, width, generator=gen).to(t).to(cuda) if kind else None
    rng = ops.rng_state(5, cuda)
    r, h, rz, rr = ops.norm_residual_fwd(z, x, w[0], w[1], gate, w[2], 0.8, 0.3, rng)
    want = ops.norm_residual_bwd(dr, dh, z, r, w[0], w[1], rz, rr, gate, w[2], 0.8, 0.3, rng)
    outs, stats = [Padded(n, d, t, cuda) for _ in range(2)], [torch.full((n + 2,), MARK, device=cuda) for _ in range(2)]
    at = gate.data_ptr() if kind else 0
    weights = (*(v.data_ptr() for v in w), 0)
    call("cg_norm_residual_fwd", z.data_ptr(), d, x.data_ptr(), d, at, width, kind, *weights, 0.8, 0.3, rng.data_ptr(), 1e-6,
         outs[0].at(), outs[0].ld, outs[1].at(), outs[1].ld, stats[0][1:].data_ptr(), stats[1][1:].data_ptr(), n, d, CODE[t])
    outs[0].check(r, "r")
    outs[1].check(h, "h")
    for got, stat in zip(stats, (rz, rr)):
        assert torch.equal(got[1:-1], stat) and got[0] == MARK and got[-1] == MARK
    dz, dx, dgate = (Padded(n, v, t, cuda) for v in (d, d, max(width, 1)))
    sums, space = [torch.full((d + 2,), MARK, device=cuda) for _ in range(3)], work("cg_norm_bwd_workspace", n, d)
    call("cg_norm_residual_bwd", dr.data_ptr(), d, dh.data_ptr(), d, z.data_ptr(), d, r.data_ptr(), d, at, width, kind, *weights,
         0.8, 0.3, rng.data_ptr(), rz.data_ptr(), rr.data_ptr(), dz.at(), dz.ld, dx.at(), dx.ld, dgate.at() if kind else 0,
         dgate.ld, *(v[1:].data_ptr() for v in sums), n, d, CODE[t], space.data_ptr(), space.numel())
    dz.check(want[0], "dz")
    dx.check(want[1], "dx")
    if kind:
        dgate.check(want[2], "dgate")
    for got, value in zip(sums, want[3:]):
        assert torch.equal(got[1:-1], value) and got[0] == MARK and got[-1] == MARK


@pytest.mark.parametrize("beta", [0.0, 1.0, -0.5])
@pytest.mark.parametrize("t", FLOATS)
def test_strided_output_of_the_wrapper(cuda, t, beta):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(1)
    g, idx = torch.randn(700, 41, generator=gen).to(t).to(cuda), torch.randint(0, 60, (700,), generator=gen).to(cuda)
    old = torch.randn(60, 41, generator=gen).to(cuda)
    out = Padded(60, 41, torch.float32, cuda, fill=old)
    assert ops.embedding_bwd(g, idx, 60, 0.5, out=out.window, beta=beta) is out.window
    out.check(ops.embedding_bwd(g, idx, 60, 0.5, out=old, beta=beta), "out")
