"""CPU restatement of the row-wise training operators in 64 bits (test infrastructure: the product never imports it).

The generator is Philox 4x32 (Salmon, Moraes, Dror, Shaw 2011) on numpy's unsigned 64-bit integers.  The gradients are
closed forms of given row statistics, with the magnitudes of the terms they sum for the tests' bounds; they are pinned to
torch's automatic differentiation of the forward functions in float64, and those to differences.
"""
from __future__ import annotations

import numpy as np
import torch

ROUNDS = 7


def philox(counter, key, rounds: int = ROUNDS):
    """The four output words (arrays broadcast together) for four counter words and two key words."""
    low = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [np.uint64(v) for v in key]
    for _ in range(rounds):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> np.uint64(32)) ^ c[1] ^ k[0], b & low, (a >> np.uint64(32)) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return c


def keep_mask(seed: int, offset: int, n: int, d: int, p: float, row0: int = 0) -> torch.Tensor:
    """bool [n, d]: which elements of rows row0 .. row0 + n - 1 stay."""
    seed, offset = seed % (1 << 64), offset % (1 << 64)
    rows = np.arange(row0, row0 + n, dtype=np.uint64)[:, None]
    blocks = np.arange((d + 3) // 4, dtype=np.uint64)[None, :]
    words = philox([blocks, rows, np.uint64(offset & 0xFFFFFFFF), np.uint64(offset >> 32)],
                   [seed & 0xFFFFFFFF, seed >> 32])
    words = np.stack(np.broadcast_arrays(*words), axis=2).reshape(n, -1)[:, :d]
    threshold = int(np.floor(p * 4294967296.0 + 0.5))
    return torch.from_numpy(np.ascontiguousarray(words >= np.uint64(threshold)))


def embedding(table: torch.Tensor, idx: torch.Tensor, scale: float) -> torch.Tensor:
    idx = idx.long()
    inside = (idx >= 0) & (idx < table.shape[0])
    return torch.where(inside[:, None], table.double()[idx.clamp(0, table.shape[0] - 1)] * scale, 0.0)


def embedding_grad(g: torch.Tensor, idx: torch.Tensor, rows: int, scale: float) -> torch.Tensor:
    idx = idx.long()
    inside = (idx >= 0) & (idx < rows)
    out = torch.zeros(rows, g.shape[1], dtype=torch.float64)
    return out.index_add_(0, idx[inside], g.double()[inside]) * scale


def rms_norm(x: torch.Tensor, w, eps: float) -> torch.Tensor:
    x = x.double()
    y = x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + eps)
    return y if w is None else y * w.double()


def norm_residual(z, x, w_post, w_pre, gate, scale, alpha, keep, inv_keep, eps):
    """(r, h) in 64 bits; `keep` is a bool mask or None."""
    u = rms_norm(z, w_post, eps)
    if gate is not None:
        u = u * torch.sigmoid(gate.double())
    if keep is not None:
        u = torch.where(keep, u * inv_keep, 0.0)
    if scale is not None:
        u = u * scale.double()
    r = x.double() + alpha * u
    return r, rms_norm(r, w_pre, eps)


def rms_norm_grad(g, x, w, rho):
    """(dx, dw, and the magnitudes of the terms each of them sums) from given statistics rho [n]."""
    g, x, rho = g.double(), x.double(), rho.double()[:, None]
    w = torch.ones(x.shape[1], dtype=torch.float64) if w is None else w.double()
    xh, t = x * rho, g * w
    dx = rho * (t - xh * (t * xh).mean(dim=1, keepdim=True))
    dx_mag = rho * (t.abs() + xh.abs() * (t * xh).abs().mean(dim=1, keepdim=True))
    return dx, (g * xh).sum(dim=0), dx_mag, (g * xh).abs().sum(dim=0)


def norm_residual_grad(dr, dh, z, r, w_post, w_pre, rho_z, rho_r, gate, scale, alpha, keep, inv_keep):
    """Gradients of norm_residual from the stored r and given statistics: {name: (value, magnitude of its terms)}."""
    n, d = z.shape
    ones = torch.ones(d, dtype=torch.float64)
    w_post, scale = (ones if w is None else w.double() for w in (w_post, scale))
    into = torch.zeros(n, d, dtype=torch.float64) if dr is None else dr.double()
    mag = into.abs()
    out = {}
    if dh is not None:
        dx, dw, dx_mag, dw_mag = rms_norm_grad(dh, r, w_pre, rho_r)
        into, mag = into + dx, mag + dx_mag
        out["dw_pre"] = (dw, dw_mag)
    else:
        out["dw_pre"] = (torch.zeros(d, dtype=torch.float64),) * 2
    out["dx"] = (into, mag)
    zh = z.double() * rho_z.double()[:, None]
    sig = torch.ones(n, 1, dtype=torch.float64) if gate is None else torch.sigmoid(gate.double())
    m = torch.ones(n, d, dtype=torch.float64) if keep is None else keep.double() * inv_keep
    D, M = into * m, mag * m
    q, q_mag = (D * sig * zh).sum(dim=0), (M * sig * zh.abs()).sum(dim=0)
    out["dw_post"] = (alpha * scale * q, abs(alpha) * scale.abs() * q_mag)
    out["dscale"] = (alpha * w_post * q, abs(alpha) * w_post.abs() * q_mag)
    c = alpha * scale * w_post
    if gate is not None:
        slope = sig * torch.sigmoid(-gate.double())  # 1 - sig would cancel
        dg, dg_mag = D * c * zh * slope, M * c.abs() * zh.abs() * slope
        if gate.shape[1] == 1 and d > 1:
            dg, dg_mag = dg.sum(dim=1, keepdim=True), dg_mag.sum(dim=1, keepdim=True)
        out["dgate"] = (dg, dg_mag)
    f, f_mag = D * c * sig, M * c.abs() * sig
    rz = rho_z.double()[:, None]
    out["dz"] = (rz * (f - zh * (f * zh).mean(dim=1, keepdim=True)),
                 rz * (f_mag + zh.abs() * (f_mag * zh.abs()).mean(dim=1, keepdim=True)))
    return out
