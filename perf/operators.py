"""Cases of the row-wise training operators: dropout, embedding lookup, rms_norm and norm_residual.

Every operator works on row-major [n, d] activations.  `run` computes it in elementary torch operations, in 32 bits and
rounded once at the end, or (where `own` is set) through the framework's entry points in cagnet_amd.ops / cagnet_amd.gcn.

The generator of the dropout masks is Philox 4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers:
as easy as 1, 2, 3; 2011): key = 64-bit seed, counter = (column // 4, row, offset low, offset high), word column % 4 of
the result belongs to the element, which is dropped when the word is below round(p * 2^32).
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LOW32 = 0xFFFFFFFF
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # hidden activations of a 4,096-vertex graph, 16 wide: launch latency decides
        dict(name="dropout_fwd_tiny", op="dropout", dir="fwd", n=4096, d=16, dtype="fp32", p=0.5),
        # input features of a 232,965-vertex graph, 602 wide (rows not a multiple of 16 bytes), both directions
        dict(name="dropout_features_both", op="dropout", dir="both", n=232_965, d=602, dtype="fp32", p=0.5),
        # half-precision activations with an odd width
        dict(name="dropout_bf16_odd_both", op="dropout", dir="both", n=65_537, d=1027, dtype="bf16", p=0.1),
        # vertex types of a small graph: a few hundred table rows, int32 indices
        dict(name="embed_fwd_tiny", op="embedding", dir="fwd", n=4096, d=16, rows=512, dtype="fp32", index="int32", skew=0.0, scale=1.0),
        # learned features of a 232,965-vertex graph, popular entries first (1/rank), a training step
        dict(name="embed_vertices_step", op="embedding", dir="step", n=232_965, d=128, rows=50_021, dtype="fp32", index="int64", skew=1.0, scale=1.0),
        # a batch of token-like indices over a large table in half precision, gradient only
        dict(name="embed_bf16_wide_bwd", op="embedding", dir="bwd", n=131_072, d=1024, rows=65_536, dtype="bf16", index="int64", skew=1.0, scale=32.0),
        # normalising a handful of feature rows (a minibatch at inference)
        dict(name="rms_fwd_few_rows", op="rms_norm", dir="fwd", n=64, d=602, dtype="fp32"),
        # pre-norm of hidden activations 128 wide, a training step
        dict(name="rms_128_step", op="rms_norm", dir="step", n=232_965, d=128, dtype="fp32"),
        # wide rows in half precision, gradient only
        dict(name="rms_bf16_wide_bwd", op="rms_norm", dir="bwd", n=16_384, d=4096, dtype="bf16"),
        # residual block around a 16-wide layer of a small graph, forward
        dict(name="residual_fwd_tiny", op="norm_residual", dir="fwd", n=4096, d=16, dtype="fp32", gate="none", scaled=True, p=0.0),
        # residual block at the feature width of a 232,965-vertex graph with a gate per vertex and dropout, a training step
        dict(name="residual_602_step", op="norm_residual", dir="step", n=232_965, d=602, dtype="fp32", gate="row", scaled=True, p=0.1),
        # wide half-precision block with a gate per element, gradient only
        dict(name="residual_bf16_bwd", op="norm_residual", dir="bwd", n=32_768, d=2560, dtype="bf16", gate="full", scaled=False, p=0.1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dropout", "embedding", "rms_norm", "norm_residual"])
    dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    d = _log_int(rng, 8, 6000)
    n = _log_int(rng, 16, max(64, min(1_000_000, 60_000_000 // d)))
    c = dict(op=op, n=n, d=d, dtype=dtype)
    if op == "dropout":
        c.update(dir=rng.choice(["fwd", "both"]), p=round(rng.uniform(0.02, 0.8), 3))
    elif op == "embedding":
        c.update(dir=rng.choice(["fwd", "bwd", "step"]), rows=_log_int(rng, 8, max(16, min(200_000, 60_000_000 // d))),
                 index=rng.choice(["int32", "int64"]), skew=rng.choice([0.0, 0.7, 1.0, 1.3]), scale=rng.choice([1.0, 0.25, 11.3]))
    elif op == "rms_norm":
        c.update(dir=rng.choice(["fwd", "bwd", "step"]))
    else:
        c.update(dir=rng.choice(["fwd", "bwd", "step"]), gate=rng.choice(["none", "row", "full"]), scaled=rng.random() < 0.5,
                 p=rng.choice([0.0, 0.1, 0.35]))
    return c


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _indices(c, gen, dev):
    """Indices into the table: rank r with probability ~ 1 / (r + 1)^skew, the ranks scattered over the table."""
    u = torch.rand(c["n"], generator=gen, device=dev, dtype=torch.float64)
    rows, s = c["rows"], c["skew"]
    if s == 0.0:
        rank = (u * rows).long()
    elif s == 1.0:
        rank = torch.exp(u * math.log(rows + 1.0)).long() - 1
    else:
        top = (rows + 1.0) ** (1.0 - s)
        rank = ((u * (top - 1.0) + 1.0) ** (1.0 / (1.0 - s))).long() - 1
    rank = rank.clamp_(0, rows - 1)
    place = torch.randperm(rows, generator=gen, device=dev)
    return place[rank].to(torch.int32 if c["index"] == "int32" else torch.int64)


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    t = DTYPES[c["dtype"]]
    n, d = c["n"], c["d"]

    def normal(*shape, like=t):
        return torch.randn(*shape, generator=gen, device=dev).to(like)

    leaf = c["dir"] == "step"

    def weight():  # a training step keeps its weights in the activations' type, the gradient-only cases in fp32
        return (1.0 + 0.2 * torch.randn(d, generator=gen, device=dev)).to(t if leaf else torch.float32)

    rng = torch.tensor([(seed * 0x9E3779B97F4A7C15 + 12345) % (1 << 62), (seed * 7919) % (1 << 40)], dtype=torch.int64, device=dev)
    s = {"case": dict(c), "rng": rng}
    if c["op"] == "dropout":
        s["x"] = normal(n, d)
        if c["dir"] == "both":
            s["g"] = normal(n, d)
    elif c["op"] == "embedding":
        s["idx"] = _indices(c, gen, dev)
        if c["dir"] != "bwd":
            s["table"] = normal(c["rows"], d).requires_grad_(leaf)
        if c["dir"] != "fwd":
            s["g"] = normal(n, d)
    elif c["op"] == "rms_norm":
        s["x"] = normal(n, d).requires_grad_(leaf)
        s["w"] = weight().requires_grad_(leaf)
        if c["dir"] != "fwd":
            s["g"] = normal(n, d)
        if c["dir"] == "bwd":
            s["rstd"] = _rstd(s["x"].float())
    else:
        s["z"] = normal(n, d).requires_grad_(leaf)
        s["w_post"], s["w_pre"] = weight().requires_grad_(leaf), weight().requires_grad_(leaf)
        s["gate"] = None if c["gate"] == "none" else normal(n, 1 if c["gate"] == "row" else d).requires_grad_(leaf)
        s["scale"] = (0.3 * weight()).detach().requires_grad_(leaf) if c["scaled"] else None
        if c["dir"] != "bwd":
            s["x"] = normal(n, d).requires_grad_(leaf)
        else:
            s["r"] = normal(n, d)
            s["rstd_z"], s["rstd_r"] = _rstd(s["z"].float()), _rstd(s["r"].float())
        if c["dir"] != "fwd":
            s["dr"], s["dh"] = normal(n, d), normal(n, d)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _mulhilo(a, m):
    prod = a * m  # modulo 2^64
    return (prod >> 32) & LOW32, prod & LOW32


def _keep(rng, n, d, p):
    """True where the element stays: Philox words in 64-bit integers."""
    dev = rng.device
    seed, off = rng[0], rng[1]
    blocks = (d + 3) // 4
    c0 = torch.arange(blocks, device=dev).expand(n, blocks)
    c1 = torch.arange(n, device=dev).unsqueeze(1).expand(n, blocks)
    c2, c3 = off & LOW32, (off >> 32) & LOW32
    k0, k1 = seed & LOW32, (seed >> 32) & LOW32
    for _ in range(7):  # the generator's rounds
        h0, l0 = _mulhilo(c0, 0xD2511F53)
        h1, l1 = _mulhilo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & LOW32, (k1 + 0xBB67AE85) & LOW32
    words = torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), dim=2).reshape(n, blocks * 4)[:, :d]
    return words >= int(math.floor(p * 4294967296.0 + 0.5))


def _rstd(x32):
    return 1.0 / torch.sqrt(x32.square().mean(dim=1) + EPS)


def _rms_grad(g, x, rho, w):
    """(dx, dw) in 32 bits of y = x rho w."""
    xh = x * rho.unsqueeze(1)
    t = g * w
    return rho.unsqueeze(1) * (t - xh * (t * xh).mean(dim=1, keepdim=True)), (g * xh).sum(dim=0)


def _plain_dropout(c, s):
    t, keep = s["x"].dtype, _keep(s["rng"], c["n"], c["d"], c["p"])
    inv = 1.0 / (1.0 - c["p"])
    out = {"y": torch.where(keep, s["x"].float() * inv, 0.0).to(t)}
    if c["dir"] == "both":
        out["dx"] = torch.where(keep, s["g"].float() * inv, 0.0).to(t)
    return out


def _plain_embedding(c, s):
    out, idx = {}, s["idx"].long()
    if c["dir"] != "bwd":
        table = s["table"].detach()
        out["y"] = (table[idx].float() * c["scale"]).to(table.dtype)
    if c["dir"] != "fwd":
        dt = torch.zeros(c["rows"], c["d"], device=idx.device).index_add_(0, idx, s["g"].float())
        out["dtable"] = (dt * c["scale"]).to(s["g"].dtype)
    return out


def _plain_rms(c, s):
    t, x, w, out = s["x"].dtype, s["x"].detach().float(), s["w"].detach().float(), {}
    rho = s["rstd"] if c["dir"] == "bwd" else _rstd(x)
    if c["dir"] != "bwd":
        out["y"] = (x * rho.unsqueeze(1) * w).to(t)
    if c["dir"] == "fwd":
        out["rstd"] = rho
    else:
        dx, dw = _rms_grad(s["g"].float(), x, rho, w)
        out["dx"], out["dw"] = dx.to(t), dw.to(s["w"].dtype)
    return out


def _plain_residual(c, s):
    t, z, out = s["z"].dtype, s["z"].detach().float(), {}
    wt, w_post, w_pre = s["w_post"].dtype, s["w_post"].detach().float(), s["w_pre"].detach().float()
    scale = s["scale"].detach().float() if c["scaled"] else torch.ones_like(w_post)
    sig = 1.0 if s["gate"] is None else torch.sigmoid(s["gate"].detach().float())
    mask = _keep(s["rng"], c["n"], c["d"], c["p"]).float() * (1.0 / (1.0 - c["p"])) if c["p"] > 0 else 1.0
    rho_z = s["rstd_z"] if c["dir"] == "bwd" else _rstd(z)
    zh = z * rho_z.unsqueeze(1)
    if c["dir"] != "bwd":
        r = s["x"].detach().float() + scale * (mask * sig * (zh * w_post))
        rho_r = _rstd(r)
        out["r"], out["h"] = r.to(t), (r * rho_r.unsqueeze(1) * w_pre).to(t)
    else:
        r, rho_r = s["r"].float(), s["rstd_r"]
    if c["dir"] == "fwd":
        out["rstd_z"], out["rstd_r"] = rho_z, rho_r
        return out
    dr, dw_pre = _rms_grad(s["dh"].float(), r.to(t).float(), rho_r, w_pre)  # backward reads the stored r
    dr = dr + s["dr"].float()
    out["dw_pre"] = dw_pre.to(wt)
    out["dx"] = dr.to(t)
    dm = dr * mask
    q = (dm * sig * zh).sum(dim=0)
    out["dw_post"] = (scale * q).to(wt)
    if c["scaled"]:
        out["dscale"] = (w_post * q).to(wt)
    e = dm * scale * w_post
    if s["gate"] is not None:
        dgate = e * zh * (sig * (1.0 - sig))
        out["dgate"] = (dgate.sum(dim=1, keepdim=True) if c["gate"] == "row" else dgate).to(t)
    f = e * sig
    out["dz"] = (rho_z.unsqueeze(1) * (f - zh * (f * zh).mean(dim=1, keepdim=True))).to(t)
    return out


PLAIN = {"dropout": _plain_dropout, "embedding": _plain_embedding, "rms_norm": _plain_rms, "norm_residual": _plain_residual}


# ---------------------------------------------------------------------------------------------------------------------
# the framework's entry points
# ---------------------------------------------------------------------------------------------------------------------
def _own(c, s):
    from cagnet_amd import gcn, ops

    if c["op"] == "dropout":
        out = {"y": ops.dropout_fwd(s["x"], c["p"], s["rng"])}
        if c["dir"] == "both":
            out["dx"] = ops.dropout_bwd(s["g"], c["p"], s["rng"])
        return out
    if c["op"] == "embedding":
        if c["dir"] == "fwd":
            return {"y": ops.embedding_fwd(s["table"], s["idx"], c["scale"])}
        if c["dir"] == "bwd":
            return {"dtable": ops.embedding_bwd(s["g"], s["idx"], c["rows"], c["scale"])}
        y = gcn.embedding(s["table"], s["idx"], c["scale"])
        return {"y": y, "dtable": torch.autograd.grad(y, s["table"], s["g"])[0]}
    if c["op"] == "rms_norm":
        if c["dir"] == "fwd":
            y, rstd = ops.rms_norm_fwd(s["x"], s["w"], EPS)
            return {"y": y, "rstd": rstd}
        if c["dir"] == "bwd":
            dx, dw = ops.rms_norm_bwd(s["g"], s["x"], s["w"], s["rstd"])
            return {"dx": dx, "dw": dw}
        y = gcn.rms_norm(s["x"], s["w"], EPS)
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["g"])
        return {"y": y, "dx": dx, "dw": dw}
    more = dict(gate=s["gate"], scale=s["scale"], p=c["p"], rng=s["rng"] if c["p"] > 0 else None)
    if c["dir"] == "fwd":
        r, h, rstd_z, rstd_r = ops.norm_residual_fwd(s["z"], s["x"], s["w_post"], s["w_pre"], eps=EPS, **more)
        return {"r": r, "h": h, "rstd_z": rstd_z, "rstd_r": rstd_r}
    if c["dir"] == "bwd":
        dz, dx, dgate, dw_post, dw_pre, dscale = ops.norm_residual_bwd(s["dr"], s["dh"], s["z"], s["r"], s["w_post"], s["w_pre"],
                                                                       s["rstd_z"], s["rstd_r"], **more)
        out = {"dz": dz, "dx": dx, "dgate": dgate, "dw_post": dw_post, "dw_pre": dw_pre, "dscale": dscale}
    else:
        r, h = gcn.norm_residual(s["z"], s["x"], s["w_post"], s["w_pre"], eps=EPS, **more)
        names = [k for k in ("z", "x", "gate", "w_post", "w_pre", "scale") if s[k] is not None]
        grads = torch.autograd.grad((r, h), [s[k] for k in names], (s["dr"], s["dh"]))
        out = {"r": r, "h": h, **{"d" + k: g for k, g in zip(names, grads)}}
    return {k: v for k, v in out.items() if v is not None}


def run(state):
    c = state["case"]
    if own:
        return _own(c, state)
    return PLAIN[c["op"]](c, state)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    n, d, size = c["n"], c["d"], 4 if c["dtype"] == "fp32" else 2
    a = n * d * size  # one activation
    fwd, bwd = c["dir"] in ("fwd", "step", "both"), c["dir"] in ("bwd", "step", "both")
    nbytes = flops = 0.0
    if c["op"] == "dropout":
        nbytes, flops = (2 * a + 16) * (fwd + bwd), n * d * (fwd + bwd)
    elif c["op"] == "embedding":
        table, idx = c["rows"] * d * size, n * (4 if c["index"] == "int32" else 8)
        nbytes = idx + (a + min(a, table) if fwd else 0) + (a + table if bwd else 0)
        flops = n * d * (fwd + bwd)
    elif c["op"] == "rms_norm":
        w, rho = 4 * d, 4 * n
        if fwd:
            nbytes, flops = nbytes + 2 * a + w + rho, flops + 4 * n * d
        if bwd:  # a step reads x again only because the row's statistics and the gradient do not meet: counted once
            nbytes, flops = nbytes + (2 * a if fwd else 3 * a + rho) + 2 * w, flops + 8 * n * d
    else:
        w, gate = 4 * d, {"none": 0, "row": n * size, "full": a}[c["gate"]]
        if fwd:
            nbytes, flops = nbytes + 4 * a + gate + 3 * w + 8 * n, flops + 12 * n * d
        if bwd:  # in a step z, the gate and r are in the forward pass's count already
            nbytes, flops = nbytes + (4 * a + gate if fwd else 6 * a + 2 * gate + 8 * n) + 6 * w, flops + 26 * n * d
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits, from the definitions: forward in double precision, gradients by automatic differentiation of it
# ---------------------------------------------------------------------------------------------------------------------
def _mask64(c, s):
    """0 or 1 / (1 - p) for every element; the generator on pairs of 16-bit halves, so that no product leaves 2^48."""
    n, d, p, dev = c["n"], c["d"], c["p"], s["rng"].device
    seed, off = (int(v) & ((1 << 64) - 1) for v in s["rng"].tolist())
    threshold = int(math.floor(p * 4294967296.0 + 0.5))
    out = torch.empty(n, d, dtype=torch.float64, device=dev)
    words = (d + 3) // 4

    def times(m, v):
        lo, hi = (v & 0xFFFF) * m, (v >> 16) * m  # v m = lo + 2^16 hi
        mid = hi + (lo >> 16)
        return mid >> 16, ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)

    step = max(1, 40_000_000 // max(1, words))
    for r0 in range(0, n, step):
        rows = torch.arange(r0, min(n, r0 + step), device=dev).repeat_interleave(words)
        ctr = [torch.arange(words, device=dev).repeat(rows.numel() // words), rows,
               torch.full_like(rows, off & LOW32), torch.full_like(rows, off >> 32)]
        for k in range(7):
            key = ((seed & LOW32) + k * 0x9E3779B9 & LOW32, (seed >> 32) + k * 0xBB67AE85 & LOW32)
            (ha, la), (hb, lb) = times(0xD2511F53, ctr[0]), times(0xCD9E8D57, ctr[2])
            ctr = [hb ^ ctr[1] ^ key[0], lb, ha ^ ctr[3] ^ key[1], la]
        block = out[r0:r0 + step]
        for j in range(4):
            if j < d:
                kept = ctr[j].reshape(-1, words)[:, :(d - j + 3) // 4] >= threshold
                block[:, j::4] = kept.double() / (1.0 - p)
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    leaf = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    fwd, out = c["dir"] != "bwd", {}

    def norm(v, w):
        return v / (v.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w

    def rho(v):
        return (v.pow(2).mean(1) + EPS).rsqrt()

    if c["op"] == "dropout":
        mask = _mask64(c, s)
        out["y"] = leaf["x"] * mask
        if c["dir"] == "both":
            out["dx"] = leaf["g"] * mask
    elif c["op"] == "embedding":
        idx = s["idx"].long()
        if fwd:
            out["y"] = leaf["table"].index_select(0, idx).mul_(c["scale"])
        if c["dir"] != "fwd":
            order = torch.argsort(idx, stable=True)
            counts = torch.bincount(idx, minlength=c["rows"])
            out["dtable"] = torch.segment_reduce(leaf["g"].index_select(0, order), "sum", lengths=counts, axis=0,
                                                 initial=0.0).mul_(c["scale"])
    elif c["op"] == "rms_norm":
        x, w = leaf["x"].requires_grad_(), leaf["w"].requires_grad_()
        y = norm(x, w)
        if fwd:
            out["y"] = y.detach()
        if c["dir"] == "fwd":
            out["rstd"] = rho(x.detach())
        else:
            out["dx"], out["dw"] = torch.autograd.grad(y, (x, w), leaf["g"])
    else:
        z, w_post, w_pre = (leaf[k].requires_grad_() for k in ("z", "w_post", "w_pre"))
        u = norm(z, w_post)
        if s["gate"] is not None:
            u = u * torch.sigmoid(leaf["gate"].requires_grad_())
        if c["p"] > 0:
            u = u * _mask64(c, s)
        if c["scaled"]:
            u = u * leaf["scale"].requires_grad_()
        if fwd:
            r = leaf["x"] + u.detach()
            rho_r = rho(r)
            out["r"], out["h"] = r, norm(r, w_pre.detach())
            if c["dir"] == "fwd":
                out["rstd_z"], out["rstd_r"] = rho(z.detach()), rho_r
            r = r.to(s["z"].dtype).double()  # backward starts from the stored residual and the statistics of the sum before its rounding
        else:
            r, rho_r = leaf["r"], rho(leaf["r"])
        if c["dir"] != "fwd":
            unit, t = r * rho_r[:, None], leaf["dh"] * w_pre.detach()
            out["dw_pre"] = (leaf["dh"] * unit).sum(0)
            into = leaf["dr"] + rho_r[:, None] * (t - unit * (t * unit).sum(1, keepdim=True) / c["d"])
            out["dx"] = into
            names = [k for k in ("z", "w_post", "gate", "scale") if s[k] is not None]
            out.update({"d" + k: g for k, g in zip(names, torch.autograd.grad(u, [leaf[k] for k in names], into))})
    return out
