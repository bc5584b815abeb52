"""The gradient of a gate far from zero, where the derivative of the sigmoid is small on both sides alike.

u = 2^-24 is a rounding of the float32 arithmetic.  e^-a: two roundings of the exponent 1.44 |a| give 2 |a| u relative to it,
the hardware's exponential 2 u.  The sigmoid s = 1 / (1 + e^-a) then is off by (2 |a| + 5) u at most, its complement (a product
with e^-a above zero, a difference from 1 of a value of at most a half below) by (4 |a| + 9) u, their product by (6 |a| + 15) u.
The other factors of a gate's term are a gradient, a normalised element (1), the weights (3) and their products (3).
"""
import pytest
import torch

from oracle import row_ops_oracle as ref

pytestmark = pytest.mark.gpu

U = 2.0**-24


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["row", "full"])
@pytest.mark.parametrize("d", [3, 41, 64, 602, 1100, 8201])  # every kind of kernel: short, partial, whole and long rows
def test_gate_gradient_far_from_zero(cuda, t, kind, d):
    from cagnet_amd import ops

    gen = torch.Generator().manual_seed(d)
    n = 33 if kind == "row" else 5
    z, x, dr = (torch.randn(n, d, generator=gen).to(t) for _ in range(3))
    w = [1 + 0.3 * torch.randn(d, generator=gen) for _ in range(2)]
    count = n if kind == "row" else n * d
    gate = torch.linspace(-40, 40, count)[torch.randperm(count, generator=gen)].reshape(n, -1).to(t)
    dev = [v.to(cuda) for v in (z, x, dr, gate, *w)]
    r, _, rz, rr = ops.norm_residual_fwd(dev[0], dev[1], dev[4], None, dev[3], dev[5], 0.8)
    got = ops.norm_residual_bwd(dev[2], None, dev[0], r, dev[4], None, rz, rr, dev[3], dev[5], 0.8)[2]
    want, mag = ref.norm_residual_grad(dr, None, z, r.cpu(), w[0], None, rz.cpu(), rr.cpu(), gate, w[1], 0.8, None, 1.0)["dgate"]
    k = 6 * gate.double().abs() + 15 + 7 + (d / 64 + 10 if kind == "row" else 0)
    half = torch.finfo(t).eps / 2
    tol = half * want.abs() + (1 + half) * k * U * mag + torch.finfo(t).smallest_normal * half
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
