"""The row-wise training operators without a GPU: the oracle is pinned to published vectors and to differences, and the
entry points refuse bad arguments before any device work."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import row_ops_oracle as ref

NULL, SIZE, OVERFLOW, UNSUPPORTED, ALIAS = 1, 2, 3, 8, 10
F32, BF16, F16 = 0, 1, 2


def _lib():
    from cagnet_amd._lib import lib

    return lib


@pytest.mark.parametrize("rounds,counter,key,want", [
    (7, [0] * 4, [0] * 2, "5f6fb709 0d893f64 4f121f81 4f730a48"),
    (10, [0] * 4, [0] * 2, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
    (10, [0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
])
def test_generator_known_answers(rounds, counter, key, want):
    got = ref.philox(counter, key, rounds)
    assert " ".join("%08x" % int(v) for v in got) == want


def test_keep_mask_is_a_function_of_row_and_column():
    whole = ref.keep_mask(-3, 1 << 40, 50, 37, 0.3)
    assert torch.equal(whole[20:30], ref.keep_mask(-3, 1 << 40, 10, 37, 0.3, row0=20))
    assert torch.equal(whole[:, :9], ref.keep_mask(-3, 1 << 40, 50, 9, 0.3))
    assert not torch.equal(whole, ref.keep_mask(-3, (1 << 40) + 1, 50, 37, 0.3))
    assert not torch.equal(whole, ref.keep_mask(-2, 1 << 40, 50, 37, 0.3))
    assert bool(ref.keep_mask(1, 1, 40, 40, 0.0).all()) and not bool(ref.keep_mask(1, 1, 40, 40, 1.0).any())


def test_keep_rate():
    """200,000 draws: the count kept is within six standard deviations of its mean."""
    for p in (0.1, 0.5, 0.9):
        kept = float(ref.keep_mask(7, 11, 400, 500, p).double().mean())
        assert abs(kept - (1 - p)) < 6 * np.sqrt(p * (1 - p) / 200_000)


def test_oracle_gradients_against_differences():
    g = torch.Generator().manual_seed(3)
    n, d = 3, 5
    z, x, gate = (torch.randn(n, d, dtype=torch.float64, generator=g).requires_grad_() for _ in range(3))
    w = [torch.randn(d, dtype=torch.float64, generator=g).requires_grad_() for _ in range(3)]
    keep = ref.keep_mask(1, 2, n, d, 0.3)
    f = lambda z, x, a, b, c, gate: ref.norm_residual(z, x, a, b, gate, c, 0.7, keep, 1 / 0.7, 1e-6)  # noqa: E731
    assert torch.autograd.gradcheck(f, (z, x, *w, gate))
    t, i = torch.randn(4, d, dtype=torch.float64, generator=g).requires_grad_(), torch.tensor([3, 0, 9, 3, -1])
    assert torch.autograd.gradcheck(lambda t: ref.embedding(t, i, 1.5), (t,))
    up = torch.randn(5, d, dtype=torch.float64, generator=g)
    grad, = torch.autograd.grad(ref.embedding(t, i, 1.5), t, up)
    assert torch.allclose(grad, ref.embedding_grad(up, i, 4, 1.5), rtol=0, atol=1e-14)


@pytest.mark.parametrize("gate_kind", ["none", "row", "full"])
@pytest.mark.parametrize("which", ["both", "r", "h"])
def test_oracle_gradient_formulas_against_automatic_differentiation(gate_kind, which):
    g = torch.Generator().manual_seed(5)
    n, d = 6, 7
    z, x, dr, dh = (torch.randn(n, d, dtype=torch.float64, generator=g) for _ in range(4))
    gate = None if gate_kind == "none" else torch.randn(n, 1 if gate_kind == "row" else d, dtype=torch.float64, generator=g)
    w_post, w_pre, scale = (torch.randn(d, dtype=torch.float64, generator=g) for _ in range(3))
    leaves = dict(z=z, x=x, w_post=w_post, w_pre=w_pre, scale=scale, **({} if gate is None else {"gate": gate}))
    for v in leaves.values():
        v.requires_grad_()
    keep = ref.keep_mask(4, 4, n, d, 0.4)
    r, h = ref.norm_residual(z, x, w_post, w_pre, gate, scale, -0.6, keep, 1 / 0.6, 1e-5)
    loss = (0.0 if which == "h" else (r * dr).sum()) + (0.0 if which == "r" else (h * dh).sum())
    want = torch.autograd.grad(loss, list(leaves.values()), allow_unused=True)
    rho = lambda v: (v.square().mean(dim=1) + 1e-5).rsqrt()  # noqa: E731
    with torch.no_grad():
        got = ref.norm_residual_grad(None if which == "h" else dr, None if which == "r" else dh, z, r, w_post, w_pre, rho(z),
                                     rho(r), gate, scale, -0.6, keep, 1 / 0.6)
    for name, value in zip(leaves, want):
        value = torch.zeros_like(leaves[name]) if value is None else value
        assert torch.allclose(got["d" + name][0], value, rtol=1e-12, atol=1e-12), name
        assert bool((got["d" + name][1] >= value.abs() * (1 - 1e-12) - 1e-13).all()), name


def test_status_codes_dropout_and_rng():
    lib, one, two = _lib(), 16, 4096  # addresses are never dereferenced: validation comes first
    assert lib.cg_rng_next(None, one, None) == NULL and lib.cg_rng_next(one, one, None) == ALIAS
    assert lib.cg_dropout(None, 0, None, 0, 0, 4, F32, 0.5, one, None) == 0          # no rows
    assert lib.cg_dropout(one, 4, two, 4, 3, 4, 7, 0.5, one, None) == UNSUPPORTED   # dtype
    assert lib.cg_dropout(one, 4, two, 4, -1, 4, F32, 0.5, one, None) == SIZE
    assert lib.cg_dropout(one, 4, two, 4, 3, 0, F32, 0.5, one, None) == SIZE
    assert lib.cg_dropout(one, 4, two, 4, 1 << 32, 4, F32, 0.5, one, None) == OVERFLOW
    assert lib.cg_dropout(one, 3, two, 4, 3, 4, F32, 0.5, one, None) == SIZE
    assert lib.cg_dropout(one, 4, None, 4, 3, 4, F32, 0.5, one, None) == NULL
    assert lib.cg_dropout(one, 4, two, 4, 3, 4, F32, 0.5, None, None) == NULL        # p > 0 without a state
    assert lib.cg_dropout(one, 4, one, 5, 3, 4, F32, 0.5, one, None) == ALIAS
    for p in (-0.1, 1.1, float("nan")):
        assert lib.cg_dropout(one, 4, two, 4, 3, 4, F32, p, one, None) == SIZE


def test_status_codes_embedding():
    lib, one, two = _lib(), 16, 4096
    size = ctypes.c_int64(-1)
    assert lib.cg_embedding_bwd_workspace(10, 4, 8, None) == NULL
    assert lib.cg_embedding_bwd_workspace(10, 0, 8, ctypes.byref(size)) == SIZE
    assert lib.cg_embedding_bwd_workspace(1 << 31, 4, 8, ctypes.byref(size)) == OVERFLOW
    assert lib.cg_embedding_bwd_workspace(10, (1 << 31) - 1, 8, ctypes.byref(size)) == OVERFLOW
    assert lib.cg_embedding_bwd_workspace(10, 4, 8, ctypes.byref(size)) == 0 and size.value > 0
    fwd = lambda t=one, ldt=8, rows=4, i=one, n=5, d=8, dt=F32, o=two, ldo=8: lib.cg_embedding_fwd(  # noqa: E731
        t, ldt, rows, i, 1, n, d, dt, 1.0, o, ldo, None)
    assert fwd(n=0) == 0 and fwd(rows=0) == SIZE and fwd(d=0) == SIZE and fwd(dt=3) == UNSUPPORTED
    assert fwd(t=None) == NULL and fwd(i=None) == NULL and fwd(o=None) == NULL and fwd(ldt=7) == SIZE
    assert fwd(ldo=7) == SIZE and fwd(o=one) == ALIAS and fwd(n=1 << 31) == OVERFLOW
    bwd = lambda g=one, ldg=8, i=one, n=5, rows=4, d=8, dt=BF16, ot=F32, o=two, ldo=8, w=two, b=1 << 20: (  # noqa: E731
        lib.cg_embedding_bwd(g, ldg, i, 1, n, rows, d, dt, ot, 1.0, 0.0, o, ldo, w, b, None))
    assert bwd(ot=F16) == UNSUPPORTED and bwd(dt=5) == UNSUPPORTED and bwd(rows=0) == SIZE and bwd(n=-1) == SIZE
    assert bwd(g=None) == NULL and bwd(o=None) == NULL and bwd(w=None) == NULL and bwd(i=None) == NULL
    assert bwd(ldg=7) == SIZE and bwd(ldo=7) == SIZE and bwd(o=one) == ALIAS and bwd(b=0) == SIZE


def test_status_codes_norms():
    lib, a, b, c, e = _lib(), 16, 4096, 8192, 16384
    size = ctypes.c_int64(-1)
    assert lib.cg_norm_bwd_workspace(10, 8, None) == NULL and lib.cg_norm_bwd_workspace(10, 0, ctypes.byref(size)) == SIZE
    assert lib.cg_norm_bwd_workspace(10, 8, ctypes.byref(size)) == 0 and size.value > 0
    fwd = lambda x=a, ldx=8, wt=F32, y=b, ldy=8, r=c, n=5, d=8, dt=F32, eps=1e-6: lib.cg_rms_norm_fwd(  # noqa: E731
        x, ldx, None, wt, y, ldy, r, n, d, dt, eps, None)
    assert fwd(n=0) == 0 and fwd(x=None) == NULL and fwd(y=None) == NULL and fwd(r=None) == NULL and fwd(y=a) == ALIAS
    assert fwd(ldx=7) == SIZE and fwd(ldy=7) == SIZE and fwd(wt=BF16) == UNSUPPORTED and fwd(dt=BF16, wt=F16) == UNSUPPORTED
    for eps in (0.0, -1.0, float("inf"), float("nan")):
        assert fwd(eps=eps) == SIZE
    bwd = lambda g=a, ldg=8, x=b, ldx=8, r=c, dx=e, ld=8, n=5, w=c, wb=1 << 20: lib.cg_rms_norm_bwd(  # noqa: E731
        g, ldg, x, ldx, None, F32, r, dx, ld, None, n, 8, F32, w, wb, None)
    assert bwd(g=None) == NULL and bwd(x=None) == NULL and bwd(r=None) == NULL and bwd(dx=None) == NULL and bwd(w=None) == NULL
    assert bwd(ldg=7) == SIZE and bwd(ldx=7) == SIZE and bwd(ld=7) == SIZE and bwd(wb=8) == SIZE and bwd(dx=a) == ALIAS
    res = lambda z=a, x=b, gate=None, ldg=0, kind=0, alpha=1.0, p=0.0, rng=None, eps=1e-6, r=c, h=e, n=5, ld=8: (  # noqa: E731
        lib.cg_norm_residual_fwd(z, ld, x, 8, gate, ldg, kind, None, None, None, F32, alpha, p, rng, eps, r, 8, h, 8, a, a, n, 8,
                                 F32, None))
    assert res(n=0) == 0 and res(z=None) == NULL and res(x=None) == NULL and res(r=None) == NULL and res(ld=7) == SIZE
    assert res(kind=3) == UNSUPPORTED and res(kind=1) == NULL and res(kind=2, gate=a, ldg=7) == SIZE
    assert res(kind=1, gate=a, ldg=0) == SIZE and res(p=0.5) == NULL and res(p=2.0, rng=a) == SIZE and res(eps=0.0) == SIZE
    assert res(alpha=float("nan")) == SIZE and res(r=a) == ALIAS and res(h=b) == ALIAS and res(r=e) == ALIAS
    grad = lambda dr=a, dh=b, z=c, r=e, gate=None, kind=0, dz=32768, dx=65536, dg=None, w=a, wb=1 << 20: (  # noqa: E731
        lib.cg_norm_residual_bwd(dr, 8, dh, 8, z, 8, r, 8, gate, 8, kind, None, None, None, F32, 1.0, 0.0, None, a, a, dz, 8,
                                 dx, 8, dg, 8, None, None, None, 5, 8, F32, w, wb, None))
    assert grad(dr=None, dh=None) == NULL and grad(z=None) == NULL and grad(w=None) == NULL and grad(wb=0) == SIZE
    assert grad(kind=2, gate=16) == NULL and grad(dx=a) == ALIAS and grad(dz=65536) == ALIAS
    assert grad(kind=2, gate=131072, dg=131072) == ALIAS


def test_python_surface_refuses_cpu_tensors_and_wrong_types():
    from cagnet_amd import gcn, ops

    x, w = torch.zeros(4, 8), torch.ones(8)
    rng = torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.dropout_fwd(x, 0.5, rng), lambda: ops.dropout_bwd(x, 0.0, None), lambda: ops.rng_next(rng),
                 lambda: ops.embedding_fwd(x, torch.zeros(3, dtype=torch.int64)),
                 lambda: ops.embedding_bwd(x, torch.zeros(4, dtype=torch.int64), 5), lambda: ops.rms_norm_fwd(x, w),
                 lambda: ops.norm_residual_fwd(x, x, w, w), lambda: gcn.dropout(x, 0.5, rng), lambda: gcn.rms_norm(x, w),
                 lambda: gcn.embedding(x, torch.zeros(2, 2, dtype=torch.int32)), lambda: gcn.norm_residual(x, x, w, w)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    with pytest.raises(TypeError, match="expected a torch.Tensor"):
        ops.dropout_fwd([1.0], 0.5, rng)
    with pytest.raises(ValueError, match="generator state"):
        gcn.train(x, w, w, 4, [], None, None, dropout_p=0.5)
    state = ops.rng_state(-5, "cpu", offset=(1 << 64) - 1)
    assert state.tolist() == [-5, -1]
    assert ops.rng_state((1 << 63) + 9, "cpu").tolist() == [-(1 << 63) + 9, 0]


def test_refusals_of_workspaces_widths_and_probabilities():
    from cagnet_amd import gcn

    lib, a, b, c, e = _lib(), 16, 4096, 8192, 16384
    size, wide = ctypes.c_int64(-1), (1 << 30) + 1
    for off in (1, 4, 8):  # a workspace that is not 16-byte aligned
        assert lib.cg_embedding_bwd(a, 8, b, 1, 5, 4, 8, F32, F32, 1.0, 0.0, c, 8, e + off, 1 << 20, None) == UNSUPPORTED
        assert lib.cg_rms_norm_bwd(a, 8, b, 8, None, F32, c, e, 8, None, 5, 8, F32, c + off, 1 << 20, None) == UNSUPPORTED
        assert lib.cg_norm_residual_bwd(a, 8, b, 8, c, 8, e, 8, None, 8, 0, None, None, None, F32, 1.0, 0.0, None, a, a, 32768, 8,
                                        65536, 8, None, 8, None, None, None, 5, 8, F32, a + off, 1 << 20, None) == UNSUPPORTED
    # rows of more elements than the norms count
    assert lib.cg_norm_bwd_workspace(1, wide, ctypes.byref(size)) == OVERFLOW
    assert lib.cg_norm_bwd_workspace(1, wide - 1, ctypes.byref(size)) == 0
    assert lib.cg_rms_norm_fwd(a, wide, None, F32, b, wide, c, 1, wide, F32, 1e-6, None) == OVERFLOW
    assert lib.cg_embedding_fwd(a, wide, 1, b, 1, 1, wide, F32, 1.0, c, wide, None) == OVERFLOW
    x = torch.zeros(4, 8)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="outside"):
            gcn.train(x, x, x, 4, [], None, None, dropout_p=p, rng=torch.zeros(2, dtype=torch.int64))
