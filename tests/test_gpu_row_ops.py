"""Row-wise training operators through the C ABI against their 64-bit restatement (oracle/row_ops_oracle.py).

Tolerances count roundings.  u = 2^-24 is a rounding of the float32 arithmetic, half(t) = eps(t) / 2 the one rounding at
a store in type t.  A value made of terms of total magnitude M by a chain of k roundings is off by at most k u M; a sum
of d terms is at most d / 64 + 10 roundings long (the shortest team that adds a row has 64 lanes, or the row is shorter
than the count added for the rest), a sum over n rows at most n / 64 + 300 (rows of a workgroup in order, then the
workgroups' sums in order, whose number stays below a thousand and that are added four or more at a time).
"""
import pytest
import torch

from oracle import row_ops_oracle as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6
FLOATS = [torch.float32, torch.bfloat16, torch.float16]


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2  # half the step of the subnormal numbers


def assert_within(got, want, mag, k, name=""):
    """|got - want| <= half |want| + k u mag, the store's rounding being of a value that is itself off by k u mag."""
    t = got.dtype
    assert got.shape == want.shape, (name, got.shape, want.shape)
    tol = half(t) * want.abs() + (1 + half(t)) * k * U * mag + tiny(t)
    off = (got.detach().cpu().double() - want).abs()
    assert bool((off <= tol).all()), f"{name}: off by {float((off - tol).max())} more than the bound, worst {float((off / tol).max())}"


def normal(gen, *shape, t=torch.float32):
    return torch.randn(*shape, generator=gen).to(t)


def strided(x, cuda, pad):
    """x on the GPU inside a wider buffer, starting `pad` elements into it."""
    if pad == 0:
        return x.to(cuda)
    wide = torch.full((x.shape[0], x.shape[1] + 2 * pad), float("nan"), dtype=x.dtype, device=cuda)
    wide[:, pad:pad + x.shape[1]] = x.to(cuda)
    return wide[:, pad:pad + x.shape[1]]


# ---------------------------------------------------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------------------------------------------------
def dropout_want(x, p, seed, off):
    """The stored value exactly: one product in float32 and one rounding."""
    if p == 0.0:
        return x
    keep = ref.keep_mask(seed, off, x.shape[0], x.shape[1], p)
    inv = torch.tensor(1.0 / (1.0 - p) if p < 1.0 else 0.0, dtype=torch.float32)
    return torch.where(keep, x.float() * inv, 0.0).to(x.dtype)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("n,d,pad", [(1, 1, 0), (3, 2, 0), (1, 5000, 0), (257, 16, 0), (300, 41, 0), (64, 602, 0), (33, 1027, 3), (5, 8, 1), (2, 7, 5)])
def test_dropout_is_exact(cuda, t, n, d, pad):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(n * 1000 + d)
    x = normal(gen, n, d, t=t)
    for p, seed, off in ((0.5, 1, 0), (0.1, -7, 1 << 33), (0.999, 1 << 62, -1)):
        rng = ops.rng_state(seed, cuda, off)
        want = dropout_want(x, p, seed, off)
        assert torch.equal(ops.dropout_fwd(strided(x, cuda, pad), p, rng).cpu(), want)
        assert torch.equal(ops.dropout_bwd(strided(x, cuda, pad), p, rng).cpu(), want)
    assert torch.equal(ops.dropout_fwd(strided(x, cuda, pad), 0.0, None).cpu(), x)
    assert not bool(ops.dropout_fwd(strided(x, cuda, pad), 1.0, ops.rng_state(1, cuda)).any())


def test_dropout_many_widths(cuda):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(0)
    rng = ops.rng_state(99, cuda, 5)
    for d in list(range(1, 40)) + [63, 64, 65, 127, 129, 255, 256, 257, 511, 513, 2047, 2049]:
        for t in (torch.float32, torch.bfloat16):
            x = normal(gen, 19, d, t=t)
            assert torch.equal(ops.dropout_fwd(x.to(cuda), 0.3, rng).cpu(), dropout_want(x, 0.3, 99, 5)), (d, t)


def test_dropout_drops_infinities_and_nan(cuda):
    from cagnet_amd import ops

    x = torch.full((40, 24), float("inf"))
    x[::2] = float("nan")
    keep = ref.keep_mask(3, 1, 40, 24, 0.5)
    got = ops.dropout_fwd(x.to(cuda), 0.5, ops.rng_state(3, cuda, 1)).cpu()
    assert bool((got[~keep] == 0).all()) and bool((~torch.isfinite(got[keep])).all())


def test_dropout_in_place_and_empty(cuda):
    from cagnet_amd import _lib, ops

    gen = torch.Generator().manual_seed(1)
    x = normal(gen, 100, 37)
    y, rng = x.to(cuda), ops.rng_state(8, cuda)
    stream = torch.cuda.current_stream().cuda_stream
    assert _lib.lib.cg_dropout(y.data_ptr(), 37, y.data_ptr(), 37, 100, 37, 0, 0.4, rng.data_ptr(), stream) == 0
    assert torch.equal(y.cpu(), dropout_want(x, 0.4, 8, 0))
    assert ops.dropout_fwd(torch.empty(0, 5, device=cuda), 0.4, rng).shape == (0, 5)


def test_rng_next_steps_the_offset_and_wraps(cuda):
    from cagnet_amd import ops

    state = ops.rng_state(12, cuda, (1 << 64) - 1)
    first, second = ops.rng_next(state), ops.rng_next(state)
    assert first.tolist() == [12, -1] and second.tolist() == [12, 0] and state.tolist() == [12, 1]


def test_dropout_beyond_32_bit_offsets(cuda):
    """2.2e9 elements: the last rows sit past 2^31 elements and 2^32 bytes."""
    from cagnet_amd import ops

    n, d = 1_100_000, 2000
    x = torch.ones(n, d, dtype=torch.bfloat16, device=cuda)
    got = ops.dropout_fwd(x, 0.25, ops.rng_state(6, cuda, 2))
    for row0 in (0, 1_073_741, n - 7):
        keep = ref.keep_mask(6, 2, 7, d, 0.25, row0=row0)
        assert torch.equal(got[row0:row0 + 7].cpu().float() != 0, keep), row0


# ---------------------------------------------------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------------------------------------------------
EMBED = [  # n, rows, d, pad
    (1, 1, 1, 0), (1, 3, 5, 0), (7, 2, 16, 0), (64, 1000, 4, 0), (300, 50, 41, 0), (5000, 17, 128, 0), (2048, 600, 602, 1),
    (2049, 70000, 8, 0), (9000, 300000, 3, 0), (4097, 1, 33, 0), (20000, 40, 257, 2), (31, 9, 4099, 0), (6000, 513, 64, 0),
    # one tile, two tiles and more tiles of indices than the scatter adds up itself; tables of one, two and three sort passes
    (4096, 1023, 2, 0), (4097, 1024, 2, 0), (300_000, 1000, 3, 0), (5000, (1 << 20) + 5, 2, 0),
]


def skewed(gen, n, rows):
    """Popular rows first, and a few indices outside the table."""
    rank = (rows ** torch.rand(n, generator=gen, dtype=torch.float64)).long() - 1
    rank[torch.rand(n, generator=gen) < 0.02] = -1
    rank[torch.rand(n, generator=gen) < 0.02] = rows
    return rank


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("n,rows,d,pad", EMBED)
def test_embedding(cuda, t, n, rows, d, pad):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(n + rows + d)
    table, g = normal(gen, rows, d, t=t), normal(gen, n, d, t=t)
    for kind, it in (("skew", torch.int64), ("flat", torch.int32), ("one", torch.int32)):
        idx = skewed(gen, n, rows) if kind == "skew" else torch.randint(0, rows, (n,), generator=gen)
        if kind == "one":
            idx = torch.full((n,), rows - 1)
        di = idx.to(it).to(cuda)
        got = ops.embedding_fwd(strided(table, cuda, pad), di, 0.7)
        want = (ref.embedding(table.float(), idx, 1.0).float() * torch.tensor(0.7, dtype=torch.float32)).to(t)
        assert torch.equal(got.cpu(), want)
        # a sum of m terms takes at most m - 1 additions one after the other, plus the product with the scale
        most = int(torch.bincount(idx[(idx >= 0) & (idx < rows)], minlength=1).max())
        want, mag = ref.embedding_grad(g, idx, rows, 0.7), ref.embedding_grad(g.abs(), idx, rows, 0.7)
        dg = strided(g, cuda, pad)
        got = ops.embedding_bwd(dg, di, rows, 0.7)
        assert got.dtype == t
        assert_within(got, want, mag, min(most, 2000) + 2, kind)
        assert torch.equal(got, ops.embedding_bwd(dg, di, rows, 0.7))
        # into float32, on top of what is there
        base = normal(gen, rows, d)
        for beta in (0.0, 1.0, -0.5):
            out = strided(base, cuda, pad)
            assert ops.embedding_bwd(dg, di, rows, 0.7, out=out, beta=beta) is out
            assert_within(out, want + beta * base.double(), mag + abs(beta) * base.double().abs(), min(most, 2000) + 4, f"{kind} {beta}")


def test_embedding_beta_zero_ignores_what_is_there(cuda):
    from cagnet_amd import ops

    out = torch.full((6, 5), float("nan"), device=cuda)
    idx = torch.tensor([4, 4, 1], device=cuda)
    ops.embedding_bwd(torch.ones(3, 5, device=cuda), idx, 6, out=out, beta=0.0)
    assert out[:, 0].tolist() == [0, 1, 0, 0, 2, 0]


def test_embedding_without_indices(cuda):
    from cagnet_amd import ops

    none = torch.empty(0, dtype=torch.int64, device=cuda)
    assert ops.embedding_fwd(torch.ones(4, 3, device=cuda), none).shape == (0, 3)
    assert not bool(ops.embedding_bwd(torch.empty(0, 3, device=cuda), none, 4).any())
    outside = torch.tensor([-1, 4, 1 << 40, -(1 << 40)], device=cuda)
    assert not bool(ops.embedding_fwd(torch.ones(4, 3, device=cuda), outside).any())
    assert not bool(ops.embedding_bwd(torch.ones(4, 3, device=cuda), outside, 4).any())


def test_embedding_rows_not_named_stay_when_accumulating(cuda):
    from cagnet_amd import ops

    out = torch.full((1000, 9), float("nan"), device=cuda)
    out[[3, 700]] = 1.0
    ops.embedding_bwd(torch.ones(5, 9, device=cuda), torch.tensor([3, 3, 700, 3, -1], device=cuda), 1000, out=out, beta=1.0)
    assert out[3, 0].item() == 4.0 and out[700, 8].item() == 2.0 and int(torch.isnan(out[:, 0]).sum()) == 998


def test_embedding_beyond_32_bit_offsets(cuda):
    """A table of 2.2e9 elements and 2.2e9 looked-up ones."""
    from cagnet_amd import ops

    rows, d = 1_100_000, 2000
    table = torch.zeros(rows, d, dtype=torch.bfloat16, device=cuda)
    table[-1] = 3.0
    table[0] = 1.0
    idx = torch.full((rows,), rows - 1, device=cuda)
    idx[::2] = 0
    out = ops.embedding_fwd(table, idx)
    assert bool((out[::2] == 1).all()) and bool((out[1::2] == 3).all())
    g = ops.embedding_bwd(out, idx, rows, out=torch.empty(rows, d, device=cuda))
    assert bool((g[0] == rows // 2).all()) and bool((g[-1] == 3 * (rows // 2)).all()) and not bool(g[1:-1].any())


# ---------------------------------------------------------------------------------------------------------------------
# norms
# ---------------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 0), (1, 2, 0), (5, 3, 0), (2, 16, 0), (700, 16, 0), (33, 41, 0), (260, 128, 0), (9, 255, 0), (40, 256, 0), (17, 260, 1),
          (50, 602, 0), (12, 1024, 0), (3, 1025, 3), (6, 2048, 0), (5, 2563, 0), (4, 4096, 0), (3, 8200, 1), (2, 16384, 0), (2, 20011, 0),
          (2500, 24, 0), (1, 602, 0),
          # several steps of every team: more rows than the workgroups of a launch hold at once, and the longest rows of each kind
          (70_000, 8, 0), (4200, 300, 0), (700, 1030, 0), (3, 5003, 1), (2, 8192, 0), (600, 8201, 0)]


def wtypes(t):
    return [torch.float32] if t == torch.float32 else [torch.float32, t]


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("n,d,pad", SHAPES)
def test_rms_norm(cuda, t, n, d, pad):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(n * 7 + d)
    x, g = normal(gen, n, d, t=t), normal(gen, n, d, t=t)
    for w in [None] + [(1 + 0.3 * normal(gen, d)).to(wt) for wt in wtypes(t)]:
        dw = None if w is None else w.to(cuda)
        y, rstd = ops.rms_norm_fwd(strided(x, cuda, pad), dw, EPS)
        want = ref.rms_norm(x, w, EPS)
        k = d / 64 + 24
        assert_within(y, want, want.abs(), k, "y")
        rho = (x.double().square().mean(dim=1) + EPS).rsqrt()
        assert_within(rstd, rho, rho, k, "rstd")
        dx, gw = ops.rms_norm_bwd(strided(g, cuda, pad), strided(x, cuda, pad), dw, rstd)
        want_dx, want_dw, mag_dx, mag_dw = ref.rms_norm_grad(g, x, w, rstd.cpu())
        assert_within(dx, want_dx, mag_dx, d / 64 + 32, "dx")
        if w is None:
            assert gw is None
        else:
            assert gw.dtype == w.dtype
            assert_within(gw, want_dw, mag_dw, n / 64 + 310, "dw")


def test_rms_norm_zero_large_and_broken_rows(cuda):
    from cagnet_amd import ops

    x = torch.zeros(5, 70)
    x[1] = 1e15
    x[2, 3] = float("nan")
    x[3] = 1e-20
    x[4] = torch.arange(70.0)
    y, rstd = (v.cpu() for v in ops.rms_norm_fwd(x.to(cuda), None, 1e-6))
    assert not bool(y[0].any()) and abs(float(rstd[0]) - 1000.0) < 1e-3
    assert torch.allclose(y[1], torch.ones(70), atol=1e-6) and bool(torch.isnan(y[2]).all())
    assert torch.allclose(y[3], torch.full((70,), 1e-17), rtol=1e-5) and bool(torch.isfinite(y[4]).all())
    dx, _ = ops.rms_norm_bwd(torch.ones(5, 70, device=cuda), x.to(cuda), None, rstd.to(cuda))
    assert torch.allclose(dx[0].cpu(), torch.full((70,), 1000.0), rtol=1e-6) and bool(torch.isnan(dx[2]).all())


def residual_inputs(gen, n, d, t, gate_kind, wt, weighted=True):
    z, x, dr, dh = (normal(gen, n, d, t=t) for _ in range(4))
    gate = None if gate_kind == "none" else normal(gen, n, 1 if gate_kind == "row" else d, t=t)
    ws = [(1 + 0.3 * normal(gen, d)).to(wt) if weighted else None for _ in range(3)]
    return z, x, dr, dh, gate, ws


def check_residual(cuda, gen, n, d, pad, t, gate_kind, wt, p, weighted=True, alpha=-0.8):
    from cagnet_amd import ops

    z, x, dr, dh, gate, (w_post, w_pre, scale) = residual_inputs(gen, n, d, t, gate_kind, wt, weighted)
    on = lambda v: None if v is None else (strided(v, cuda, pad) if v.dim() == 2 else v.to(cuda))  # noqa: E731
    rng = ops.rng_state(21, cuda, 4) if p > 0 else None
    more = dict(gate=on(gate), scale=on(scale), alpha=alpha, p=p, rng=rng)
    r, h, rstd_z, rstd_r = ops.norm_residual_fwd(on(z), on(x), on(w_post), on(w_pre), eps=EPS, **more)
    keep = ref.keep_mask(21, 4, n, d, p) if p > 0 else None
    inv = 1 / (1 - p)
    want_r, want_h = ref.norm_residual(z, x, w_post, w_pre, gate, scale, alpha, keep, inv, EPS)
    # r sums x and u; what it is off by reaches h directly and through the statistics of the row
    k = d / 64 + 34
    parts = x.double().abs() + (want_r - x.double()).abs()
    assert_within(r, want_r, parts, k, "r")
    rho_r = (want_r.square().mean(dim=1, keepdim=True) + EPS).rsqrt()
    spread = (parts.square().mean(dim=1, keepdim=True) + EPS).sqrt() * rho_r
    w = torch.ones(d, dtype=torch.float64) if w_pre is None else w_pre.double()
    assert_within(h, want_h, parts * rho_r * w.abs() + want_h.abs() * spread, k + d / 64 + 16, "h")
    rho_z = (z.double().square().mean(dim=1) + EPS).rsqrt()
    assert_within(rstd_z, rho_z, rho_z, d / 64 + 24, "rstd_z")
    assert_within(rstd_r, rho_r[:, 0], rho_r[:, 0] * spread[:, 0], 2 * d / 64 + 50, "rstd_r")
    for a, b in ((dr, dh), (dr, None), (None, dh)):
        got = dict(zip(("dz", "dx", "dgate", "dw_post", "dw_pre", "dscale"),
                       ops.norm_residual_bwd(on(a), on(b), on(z), strided(r.cpu(), cuda, pad), on(w_post), on(w_pre), rstd_z, rstd_r, **more)))
        want = ref.norm_residual_grad(a, b, z, r.cpu(), w_post, w_pre, rstd_z.cpu(), rstd_r.cpu(), gate, scale, alpha, keep, inv)
        for name, value in got.items():
            if value is None:
                assert name == "dgate" and gate is None or not weighted and name[1:] in ("w_post", "w_pre", "scale")
                continue
            by_row = name in ("dw_post", "dw_pre", "dscale")
            assert_within(value, *want[name], (n / 64 + 350 if by_row else d / 64 + 56) + d / 64, name)
            if by_row:
                assert value.dtype == wt


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("gate_kind", ["none", "row", "full"])
@pytest.mark.parametrize("n,d,pad", SHAPES)
def test_norm_residual(cuda, t, gate_kind, n, d, pad):
    gen = torch.Generator().manual_seed(n * 11 + d)
    for wt in wtypes(t):
        check_residual(cuda, gen, n, d, pad, t, gate_kind, wt, 0.0 if wt == torch.float32 and n % 2 else 0.3)


@pytest.mark.parametrize("p,weighted", [(0.0, True), (0.3, False), (1.0, True)])
def test_norm_residual_without_weights_and_with_everything_dropped(cuda, p, weighted):
    gen = torch.Generator().manual_seed(17)
    if p < 1.0:
        check_residual(cuda, gen, 37, 100, 0, torch.float32, "row", torch.float32, p, weighted)
        return
    from cagnet_amd import ops

    z, x, dr, dh, gate, ws = residual_inputs(gen, 37, 100, torch.float32, "full", torch.float32)
    z, x, dr, dh, gate, w_post, w_pre, scale = (v.to(cuda) for v in (z, x, dr, dh, gate, *ws))
    rng = ops.rng_state(1, cuda)
    r, h, rz, rr = ops.norm_residual_fwd(z, x, w_post, w_pre, gate, scale, p=1.0, rng=rng)
    assert torch.equal(r, x)
    dz, dx, dgate, dwp, _, ds = ops.norm_residual_bwd(dr, dh, z, r, w_post, w_pre, rz, rr, gate, scale, p=1.0, rng=rng)
    assert not any(bool(v.any()) for v in (dz, dgate, dwp, ds)) and bool(dx.any())


def test_norms_of_no_rows(cuda):
    from cagnet_amd import ops

    x, w = torch.empty(0, 12, device=cuda), torch.ones(12, device=cuda)
    s = torch.empty(0, device=cuda)
    y, rstd = ops.rms_norm_fwd(x, w)
    assert y.shape == (0, 12) and rstd.shape == (0,)
    dx, dw = ops.rms_norm_bwd(x, x, w, s)
    assert dx.shape == (0, 12) and not bool(dw.any())
    r, h, _, _ = ops.norm_residual_fwd(x, x, w, w, x, w)
    out = ops.norm_residual_bwd(r, h, x, r, w, w, s, s, x, w)
    assert out[0].shape == (0, 12) and not any(bool(v.any()) for v in out[3:])


def test_norm_gate_extremes(cuda):
    """Gates far out on either side: the sigmoid is 0 or 1 and its gradient 0, never NaN."""
    from cagnet_amd import ops

    z = torch.randn(4, 33, generator=torch.Generator().manual_seed(0)).to(cuda)
    gate = torch.tensor([[-float("inf")], [float("inf")], [-200.0], [200.0]], device=cuda)
    r, h, rz, rr = ops.norm_residual_fwd(z, torch.zeros_like(z), None, None, gate)
    assert not bool(r[0].any()) and not bool(r[2].any()) and bool(r[1].all()) and bool(r[3].all())
    out = ops.norm_residual_bwd(z, None, z, r, None, None, rz, rr, gate)
    assert out[2].flatten().tolist() == [0.0] * 4 and all(bool(torch.isfinite(v).all()) for v in out[:2])


def test_dropped_elements_of_a_broken_block_leave_the_residual(cuda):
    """A block output with NaN: its dropped elements add nothing, in both directions."""
    from cagnet_amd import ops

    z = torch.randn(6, 50, generator=torch.Generator().manual_seed(1))
    z[2, 7] = float("nan")
    x = torch.randn(6, 50, generator=torch.Generator().manual_seed(2))
    keep = ref.keep_mask(3, 9, 6, 50, 0.5)
    rng = ops.rng_state(3, cuda, 9)
    r, _, rz, rr = ops.norm_residual_fwd(z.to(cuda), x.to(cuda), None, None, p=0.5, rng=rng)
    assert torch.equal(r.cpu()[~keep], x[~keep]) and bool(torch.isnan(r.cpu()[2][keep[2]]).all())
    assert bool(torch.isfinite(r[[0, 1, 3, 4, 5]]).all())
    dr = torch.full((6, 50), float("inf"))
    dr[keep] = 1.0
    out = ops.norm_residual_bwd(dr.to(cuda), None, z.to(cuda), r, None, None, rz, rr, p=0.5, rng=rng)
    assert bool(torch.isfinite(out[0][[0, 1, 3, 4, 5]]).all())  # infinite gradients of dropped elements do not reach z


def test_norms_repeat_bit_for_bit(cuda):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(2)
    z, x, dr, dh, gate, ws = residual_inputs(gen, 5000, 130, torch.float32, "full", torch.float32)
    z, x, dr, dh, gate, w_post, w_pre, scale = (v.to(cuda) for v in (z, x, dr, dh, gate, *ws))
    rng = ops.rng_state(5, cuda)
    run = lambda: (lambda f: f + ops.norm_residual_bwd(dr, dh, z, f[0], w_post, w_pre, f[2], f[3], gate, scale, p=0.2, rng=rng))(  # noqa: E731
        ops.norm_residual_fwd(z, x, w_post, w_pre, gate, scale, p=0.2, rng=rng))
    assert all(torch.equal(a, b) for a, b in zip(run(), run()))


def test_fused_dropout_uses_the_masks_of_dropout(cuda):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(9)
    z = (normal(gen, 90, 77).abs() + 0.1).to(cuda)
    rng = ops.rng_state(-4, cuda, 1 << 50)
    r, _, _, _ = ops.norm_residual_fwd(z, torch.zeros_like(z), None, None, p=0.35, rng=rng)
    assert torch.equal(r != 0, ops.dropout_fwd(z, 0.35, rng) != 0)


def test_norm_beyond_32_bit_offsets(cuda):
    from cagnet_amd import ops

    n, d = 1_100_000, 2000
    x = torch.ones(n, d, dtype=torch.bfloat16, device=cuda)
    x[-1] = 2.0
    w = torch.full((d,), 0.5, device=cuda)
    y, rstd = ops.rms_norm_fwd(x, w)
    assert abs(float(rstd[-1]) - 0.5) < 1e-6 and bool((y == 0.5).all())
    dx, dw = ops.rms_norm_bwd(y, x, w, rstd)
    assert abs(float(dw[0]) / (0.5 * n) - 1) < 1e-4 and float(dx.abs().max()) < 1e-2


# ---------------------------------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------------------------------
def test_refusals(cuda):
    from cagnet_amd import gcn, ops

    x, w, rng = torch.ones(4, 8, device=cuda), torch.ones(8, device=cuda), ops.rng_state(1, cuda)
    i = torch.zeros(4, dtype=torch.int64, device=cuda)
    for error, match, call in [
        (TypeError, "float32, bfloat16 or float16", lambda: ops.dropout_fwd(x.double(), 0.5, rng)),
        (ValueError, "2 dimensions", lambda: ops.dropout_fwd(x[0], 0.5, rng)),
        (ValueError, "no elements", lambda: ops.dropout_fwd(x[:, :0], 0.5, rng)),
        (ValueError, "generator state", lambda: ops.dropout_fwd(x, 0.5, None)),
        (ValueError, "generator state", lambda: ops.dropout_fwd(x, 0.5, rng.repeat(2))),
        (TypeError, "int64", lambda: ops.dropout_fwd(x, 0.5, rng.int())),
        (ValueError, "outside", lambda: ops.dropout_fwd(x, 1.5, rng)),
        (ValueError, "outside", lambda: ops.dropout_fwd(x, float("nan"), rng)),
        (TypeError, "int32 or int64", lambda: ops.embedding_fwd(x, i.float())),
        (ValueError, "1 dimension", lambda: ops.embedding_fwd(x, i[None])),
        (ValueError, "on cpu", lambda: ops.embedding_fwd(x, i.cpu())),
        (ops.CagnetError, "CG_ERR_SIZE", lambda: ops.embedding_fwd(x[:0], i)),
        (ValueError, "entries", lambda: ops.embedding_bwd(x, i[:2], 3)),
        (ops.CagnetError, "CG_ERR_SIZE", lambda: ops.embedding_bwd(x, i, 0)),
        (ops.CagnetError, "CG_ERR_SIZE", lambda: ops.embedding_bwd(x, i, -3)),
        (TypeError, "dtype", lambda: ops.embedding_bwd(x, i, 4, out=x.half())),
        (ValueError, "shape", lambda: ops.embedding_bwd(x, i, 5, out=x)),
        (ValueError, "row-major", lambda: ops.embedding_bwd(x, i, 8, out=torch.ones(8, 8, device=cuda).t())),
        (ops.CagnetError, "CG_ERR_ALIAS", lambda: ops.embedding_bwd(x, i, 4, out=x)),
        (TypeError, "weight", lambda: ops.rms_norm_fwd(x, w.half())),
        (ValueError, "weight", lambda: ops.rms_norm_fwd(x, w[:7])),
        (ops.CagnetError, "eps", lambda: ops.rms_norm_fwd(x, w, 0.0)),
        (ValueError, "shape", lambda: ops.rms_norm_bwd(x[:3], x, w, w[:4])),
        (ValueError, "rstd", lambda: ops.rms_norm_bwd(x, x, w, w[:3])),
        (TypeError, "x: expected dtype", lambda: ops.norm_residual_fwd(x, x.half(), w, w)),
        (TypeError, "share a dtype", lambda: ops.norm_residual_fwd(x.half(), x.half(), w, w.half())),
        (ValueError, "gate", lambda: ops.norm_residual_fwd(x, x, w, w, gate=x[:, :3])),
        (ValueError, "gate", lambda: ops.norm_residual_fwd(x, x, w, w, gate=x[:1])),
        (TypeError, "gate", lambda: ops.norm_residual_fwd(x, x, w, w, gate=x[:, :1].half())),
        (ops.CagnetError, "alpha", lambda: ops.norm_residual_fwd(x, x, w, w, alpha=float("inf"))),
        (ValueError, "at least one", lambda: ops.norm_residual_bwd(None, None, x, x, w, w, w[:4], w[:4])),
        (ValueError, "generator state", lambda: gcn.norm_residual(x, x, w, w, p=0.1)),
    ]:
        with pytest.raises(error, match=match):
            call()


def test_a_stepped_state_is_refused_in_backward(cuda):
    from cagnet_amd import gcn

    state = gcn.rng_state(3, cuda)
    y = gcn.dropout(torch.ones(4, 4, device=cuda, requires_grad=True), 0.5, state)  # the state itself, not a snapshot
    gcn.rng_next(state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---------------------------------------------------------------------------------------------------------------------
# together, as a training step uses them
# ---------------------------------------------------------------------------------------------------------------------
def deep_problem(cuda, n_scale=7, d=24, classes=5, types=9, seed=0):
    from cagnet_amd import ops
    from tests.util import small_graph

    row, col, val, n = small_graph(n_scale, 600, seed)
    gen = torch.Generator().manual_seed(seed)
    par = {"table": normal(gen, types, d), "w0": 1 + 0.1 * normal(gen, d), "out": normal(gen, d, classes) * 0.3}
    for k in (1, 2):
        par.update({f"W{k}": normal(gen, d, d) * 0.3, f"post{k}": 1 + 0.1 * normal(gen, d), f"pre{k}": 1 + 0.1 * normal(gen, d),
                    f"scale{k}": 0.5 + 0.1 * normal(gen, d), f"gate{k}": normal(gen, n, 1)})
    idx, y = torch.randint(-1, types, (n,), generator=gen), torch.randint(0, classes, (n,), generator=gen)
    blk = ops.CsrMatrix(row.int().to(cuda), col.int().to(cuda), val.to(cuda), n, n, transpose=True)
    A = torch.sparse_coo_tensor(torch.stack([row, col]), val.double(), (n, n)).to_dense()
    return par, idx, y, blk, A, n, d


def deep_loss(par, idx, y, blk, n, state):
    """Embedding -> dropout -> two pre-normed GCN layers with gated residual sums -> classes, and the loss."""
    import torch.nn.functional as F

    from cagnet_amd import gcn

    x = gcn.dropout(gcn.embedding(par["table"], idx, 2.0), 0.2, gcn.rng_next(state))
    h = gcn.rms_norm(x, par["w0"], EPS)
    for k in (1, 2):
        z = gcn.GCNFunc.apply(h, par[f"W{k}"], n, [blk], 0, 1, None, F.relu)
        x, h = gcn.norm_residual(z, x, par[f"post{k}"], par[f"pre{k}"], par[f"gate{k}"], par[f"scale{k}"], 0.9, 0.3,
                                 gcn.rng_next(state), EPS)
    out = gcn.GCNFunc.apply(h, par["out"], n, [blk], 0, 1, None, F.log_softmax)
    return gcn.masked_nll_loss(out, y, None)


def deep_loss64(par, idx, y, A, n, d, seed, offset):
    x = ref.embedding(par["table"], idx, 2.0)
    x = torch.where(ref.keep_mask(seed, offset, n, d, 0.2), x / 0.8, 0.0)
    h = ref.rms_norm(x, par["w0"], EPS)
    for k in (1, 2):
        z = torch.relu(A @ h @ par[f"W{k}"])
        x, h = ref.norm_residual(z, x, par[f"post{k}"], par[f"pre{k}"], par[f"gate{k}"], par[f"scale{k}"], 0.9,
                                 ref.keep_mask(seed, offset + k, n, d, 0.3), 1 / 0.7, EPS)
    return torch.nn.functional.nll_loss(torch.log_softmax(A @ h @ par["out"], 1), y)


def test_deep_step_against_64_bits_and_differences(cuda):
    from cagnet_amd import gcn

    par, idx, y, blk, A, n, d = deep_problem(cuda)
    dev = {k: v.to(cuda).requires_grad_() for k, v in par.items()}
    state = gcn.rng_state(77, cuda, 10)
    loss = deep_loss(dev, idx.to(cuda), y.to(cuda), blk, n, state)
    loss.backward()
    assert state.tolist() == [77, 13]
    p64 = {k: v.double().requires_grad_() for k, v in par.items()}
    want = deep_loss64(p64, idx, y, A, n, d, 77, 10)
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5
    gen = torch.Generator().manual_seed(1)
    for k in par:
        off = float((dev[k].grad.cpu().double() - p64[k].grad).abs().max())
        # the whole-step bound of the framework's other tests: 2e-4 of the largest entry
        assert off <= 2e-4 * max(float(p64[k].grad.abs().max()), 1e-3), (k, off)
        # and along a random direction against a central difference of the 64-bit loss: ReLU kinks within the step and its
        # third derivative stay below 1e-3 of the slope's scale
        v = torch.randn(par[k].shape, generator=gen, dtype=torch.float64)
        step = 1e-6
        with torch.no_grad():
            f = lambda s: float(deep_loss64({**p64, k: p64[k].detach() + s * step * v}, idx, y, A, n, d, 77, 10))  # noqa: E731
            slope = (f(1) - f(-1)) / (2 * step)
        got = float((dev[k].grad.cpu().double() * v).sum())
        assert abs(got - slope) <= 1e-3 * float((p64[k].grad.abs() * v.abs()).sum()) + 1e-7, k


def test_deep_step_captured_and_replayed(cuda):
    """One graph of forward and backward: every replay draws new masks and equals the eager step at the same state."""
    from cagnet_amd import gcn

    par, idx, y, blk, A, n, d = deep_problem(cuda, seed=3)
    dev = {k: v.to(cuda).requires_grad_() for k, v in par.items()}
    di, dy, leaves = idx.to(cuda), y.to(cuda), list(dev.values())

    def step(state):
        loss = deep_loss(dev, di, dy, blk, n, state)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):  # the products and the loss need one eager call on the stream first
        step(gcn.rng_state(1, cuda))
    torch.cuda.synchronize()
    state = gcn.rng_state(50, cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step(state)
    losses = []
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in out]
        want = step(gcn.rng_state(50, cuda, 3 * k))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k
        losses.append(float(got[0]))
    assert len(set(losses)) == 4 and state.tolist() == [50, 12]


def test_operators_capture_without_a_first_eager_call_and_graphs_do_not_share_workspaces(cuda):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(4)
    graphs = []
    for n in (3000, 4100):
        g, w = normal(gen, n, 36).to(cuda), torch.ones(36, device=cuda)
        x, idx = normal(gen, n, 36).to(cuda), torch.randint(0, 700, (n,), generator=gen).to(cuda)
        rstd = torch.ones(n, device=cuda)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = (ops.embedding_bwd(g, idx, 700), *ops.rms_norm_bwd(g, x, w, rstd))
        graphs.append((graph, out, (g, idx, x, w, rstd), torch.cuda.Stream()))
    for _ in range(3):
        for graph, _, _, stream in graphs:  # side by side on two streams
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, (g, idx, x, w, rstd), _ in graphs:
            want = (ops.embedding_bwd(g, idx, 700), *ops.rms_norm_bwd(g, x, w, rstd))
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            for v in out:
                v.zero_()


def test_on_another_stream(cuda):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(6)
    x, idx = normal(gen, 50_000, 64).to(cuda), torch.randint(0, 999, (50_000,), generator=gen).to(cuda)
    want = (ops.embedding_bwd(x, idx, 999), ops.rms_norm_fwd(x, None)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = (ops.embedding_bwd(x, idx, 999), ops.rms_norm_fwd(x, None)[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("shape", [(6,), (2, 3), (2, 1, 3), ()])
def test_embedding_of_any_shape(cuda, shape):
    from cagnet_amd import gcn

    gen = torch.Generator().manual_seed(8)
    table = normal(gen, 7, 10).to(cuda).requires_grad_()
    idx = torch.randint(0, 7, shape, generator=gen).to(cuda)
    out = gcn.embedding(table, idx, 3.0)
    assert out.shape == (*shape, 10) and torch.equal(out, table[idx] * 3.0)
    out.backward(torch.ones_like(out))
    want = torch.zeros(7, 10, device=cuda).index_add_(0, idx.reshape(-1), torch.full((idx.numel(), 10), 3.0, device=cuda))
    assert torch.equal(table.grad, want)


def test_nodes_without_some_gradients(cuda):
    """Frozen weights, an unused output, and broadcast incoming gradients (a sum's)."""
    from cagnet_amd import gcn

    gen = torch.Generator().manual_seed(12)
    z, x = normal(gen, 9, 14).to(cuda).requires_grad_(), normal(gen, 9, 14).to(cuda)
    r, h = gcn.norm_residual(z, x, None, torch.ones(14, device=cuda))
    h.sum().backward()  # r is not used
    z64 = z.detach().cpu().double().requires_grad_()
    ref.norm_residual(z64, x.cpu(), None, None, None, None, 1.0, None, 1.0, EPS)[1].sum().backward()
    assert torch.allclose(z.grad.cpu().double(), z64.grad, atol=1e-5)
    z.grad = None
    gcn.norm_residual(z, x, None, None)[0].sum().backward()  # h is not used
    z64.grad = None
    ref.norm_residual(z64, x.cpu(), None, None, None, None, 1.0, None, 1.0, EPS)[0].sum().backward()
    assert torch.allclose(z.grad.cpu().double(), z64.grad, atol=1e-5)


# ---------------------------------------------------------------------------------------------------------------------
# dropout in gcn.train
# ---------------------------------------------------------------------------------------------------------------------
def train_problem(cuda):
    import types

    from cagnet_amd import ops, synth

    p = synth.make_problem(scale=8, n_edges=1500, features=20, hidden=16, classes=6, mask_fraction=0.6, seed=2)
    blk = ops.CsrMatrix(p.row.int().to(cuda), p.col.int().to(cuda), p.val.to(cuda), p.n, p.n, transpose=True)
    data = types.SimpleNamespace(y=p.y.to(cuda), train_mask=p.train_mask.to(cuda))
    return p, blk, data


def test_train_with_dropout_against_64_bits(cuda):
    from cagnet_amd import gcn

    p, blk, data = train_problem(cuda)
    w1, w2 = (w.to(cuda).requires_grad_() for w in (p.w1, p.w2))
    state = gcn.rng_state(9, cuda)
    opt = torch.optim.SGD([w1, w2], lr=0.1)
    A = torch.sparse_coo_tensor(torch.stack([p.row, p.col]), p.val.double(), (p.n, p.n)).to_dense()
    m1, m2 = (w.double().clone().requires_grad_() for w in (p.w1, p.w2))
    for epoch in range(3):
        gcn.train(p.x.to(cuda).requires_grad_(), w1, w2, p.n, [blk], opt, data, dropout_p=0.5, rng=state)
        hidden = torch.relu(A @ p.x.double() @ m1)
        hidden = torch.where(ref.keep_mask(9, epoch, *hidden.shape, 0.5), hidden * 2, 0.0)
        out = torch.log_softmax(A @ hidden @ m2, 1)
        mask = p.train_mask.bool()
        loss = torch.nn.functional.nll_loss(out[mask], p.y[mask])
        assert abs(float(gcn.train.last_loss) - float(loss.detach())) <= 1e-4
        g1, g2 = torch.autograd.grad(loss, (m1, m2))
        with torch.no_grad():
            m1 -= 0.1 * g1
            m2 -= 0.1 * g2
    for a, b in ((w1, m1), (w2, m2)):
        assert float((a.detach().cpu().double() - b.detach()).abs().max()) <= 2e-4 * float(b.detach().abs().max())


def test_graphed_train_with_dropout_equals_eager(cuda):
    from cagnet_amd import gcn

    p, blk, data = train_problem(cuda)

    def fresh():
        w1, w2 = (w.to(cuda).requires_grad_() for w in (p.w1, p.w2))
        return p.x.to(cuda).requires_grad_(), w1, w2, torch.optim.SGD([w1, w2], lr=0.05), gcn.rng_state(4, cuda)

    x, w1, w2, opt, state = fresh()
    losses = []
    for _ in range(8):
        gcn.train(x, w1, w2, p.n, [blk], opt, data, dropout_p=0.4, rng=state)
        x.grad = None
        losses.append(float(gcn.train.last_loss))
    x, g1, g2, opt, state = fresh()
    graphed = gcn.GraphedTrain(x, g1, g2, p.n, [blk], opt, data, warmup=3, dropout_p=0.4, rng=state)
    for k in range(5):
        graphed.step()
        torch.cuda.synchronize()
        assert abs(float(graphed.loss) - losses[3 + k]) <= 1e-5, k
        torch.zeros(1000, device=cuda).sum().item()  # eager work between replays
    assert torch.allclose(g1, w1, atol=1e-5) and torch.allclose(g2, w2, atol=1e-5)
    assert state.tolist() == [4, 8]
    graphed.close()


@pytest.mark.parametrize("op", ["dropout", "embedding", "rms_norm", "norm_residual"])
def test_second_derivatives_are_refused_first_ones_are_the_same(cuda, op):
    from cagnet_amd import gcn, ops

    gen = torch.Generator(device="cuda").manual_seed(5)
    x, z = (torch.randn(33, 20, device="cuda", generator=gen).requires_grad_() for _ in range(2))
    w = torch.randn(20, device="cuda", generator=gen).requires_grad_()
    g = torch.randn(33, 20, device="cuda", generator=gen).requires_grad_()
    idx = torch.randint(0, 33, (33,), device="cuda", generator=gen)
    rng = ops.rng_state(3)
    call, leaf = {"dropout": (lambda: gcn.dropout(x, 0.3, rng), x), "embedding": (lambda: gcn.embedding(x, idx, 2.0), x),
                  "rms_norm": (lambda: gcn.rms_norm(x, w), x),
                  "norm_residual": (lambda: gcn.norm_residual(z, x, w, w, p=0.3, rng=rng)[1], z)}[op]
    (want,) = torch.autograd.grad(call(), leaf, g)
    (got,) = torch.autograd.grad(call(), leaf, g, create_graph=True)
    assert not want.requires_grad and torch.equal(got, want)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        got.sum().backward()


@pytest.mark.parametrize("n, d", [(1, 24), (7, 1), (1, 1), (6, 24)])
def test_results_are_contiguous_whatever_the_strides(cuda, n, d):
    from cagnet_amd import ops

    wide = torch.randn(d, 3 * n, device="cuda").t()[::3]      # columns apart, rows apart
    apart = torch.randn(n, 40, device="cuda")[:, :d]          # rows apart
    w = torch.randn(d, device="cuda")
    for x in (wide, apart):
        y, rstd = ops.rms_norm_fwd(x, w)
        dx, _ = ops.rms_norm_bwd(x, x, w, rstd)
        r, h, rz, rr = ops.norm_residual_fwd(x, x, w, w, gate=x)
        outs = [ops.dropout_fwd(x, 0.0, None), y, dx, r, h, *ops.norm_residual_bwd(x, x, x, r, w, w, rz, rr, gate=x)[:3]]
        assert all(o.is_contiguous() and o.shape == x.shape for o in outs)
        x = x.contiguous()
        y2, rstd = ops.rms_norm_fwd(x, w)
        r2, h2, rz, rr = ops.norm_residual_fwd(x, x, w, w, gate=x)
        same = [x, y2, ops.rms_norm_bwd(x, x, w, rstd)[0], r2, h2,
                *ops.norm_residual_bwd(x, x, x, r2, w, w, rz, rr, gate=x)[:3]]
        assert all(torch.equal(a, b) for a, b in zip(outs, same))


@pytest.mark.parametrize("beta", [0.0, 1.0, 0.5])
@pytest.mark.parametrize("t, d", [(torch.float32, 3), (torch.float32, 13), (torch.float32, 64), (torch.float32, 70),
                                  (torch.bfloat16, 5), (torch.bfloat16, 55), (torch.float16, 261), (torch.float16, 600)])
def test_embedding_many_hot_rows(cuda, t, d, beta):
    # every table row but the last ten has about 100 positions, row 7 a third of all; the first index is padding
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(d)
    n, rows = 60_000, 410
    idx = torch.randint(0, rows - 10, (n,), generator=gen)
    idx[torch.rand(n, generator=gen) < 1 / 3] = 7
    idx[0] = rows
    g, old = torch.randn(n, d, generator=gen).to(t), torch.randn(rows, d, generator=gen).to(t)
    out = old.to(cuda)
    ops.embedding_bwd(g.to(cuda), idx.to(cuda), rows, 0.5, out=out, beta=beta)
    want, size = torch.zeros(rows + 1, d, dtype=torch.float64), torch.zeros(rows + 1, d, dtype=torch.float64)
    want.index_add_(0, idx, g.double()), size.index_add_(0, idx, g.double().abs())
    want, size = (0.5 * want + beta * torch.cat([old, old[:1]]).double())[:rows], (0.5 * size)[:rows] + beta * old.double().abs()
    # a sum of k terms in float32 in any order is off by (k - 1) 2^-24 of their size at most; + scale, beta and the sum
    count = torch.bincount(idx, minlength=rows + 1)[:rows, None].double()
    bound = (count + 4) * 2.0**-24 * size
    bound = bound + (torch.finfo(t).eps / 2) * (want.abs() + bound) + torch.finfo(t).smallest_normal
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
