"""Cases of the residual feed-forward block's operators: layer normalisation, dropout from a counter-based generator and
the gated feed-forward product, each with its backward pass.

``run`` with ``own`` false computes them in plain torch operations in 32 bits; with ``own`` true it makes the calls that
a user of the package makes."""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5
M0, M1 = 0xD2511F53, 0xCD9E8D57      # Philox4x32 multipliers and Weyl increments (Salmon et al., 2011)
W0, W1 = 0x9E3779B9, 0xBB67AE85
MASK = 0xFFFFFFFF


# ---- cases -----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one time step of a batch of 32 sequences at the language model's width, evaluation: latency
        {"name": "ln_step", "op": "ln", "rows": 32, "dim": 650, "dtype": "fp32", "wide_w": False, "train": False},
        # one truncated-BPTT window (35 x 32 tokens) of the 2 x 650 language model, training
        {"name": "ln_window", "op": "ln", "rows": 1120, "dim": 650, "dtype": "fp32", "wide_w": False, "train": True},
        # a large training batch, larger than L2
        {"name": "ln_large", "op": "ln", "rows": 16384, "dim": 4096, "dtype": "bf16", "wide_w": False, "train": True},
        # odd width and row count (rows not 16-byte aligned), 32-bit parameters next to 16-bit activations
        {"name": "ln_odd", "op": "ln", "rows": 3001, "dim": 1027, "dtype": "fp16", "wide_w": True, "train": True},
        # dropout on the window's activations, the language model's rate
        {"name": "drop_window", "op": "drop", "rows": 1120, "dim": 650, "dtype": "fp32", "p": 0.4, "site": 1,
         "residual": False, "train": True},
        # dropout and the residual sum at the end of a block, large training batch
        {"name": "drop_large", "op": "drop", "rows": 16384, "dim": 4096, "dtype": "bf16", "p": 0.1, "site": 3,
         "residual": True, "train": True},
        # odd number of elements
        {"name": "drop_odd", "op": "drop", "rows": 3001, "dim": 1027, "dtype": "fp16", "p": 0.35, "site": 0,
         "residual": False, "train": True},
        # a single token through the block: both weight matrices are read once
        {"name": "ffn_token", "op": "ffn", "rows": 1, "dim": 2048, "hidden": 8192, "dtype": "bf16", "act": "silu",
         "train": False},
        # one time step of 32 sequences at the language model's width, evaluation
        {"name": "ffn_step", "op": "ffn", "rows": 32, "dim": 650, "hidden": 2600, "dtype": "fp32", "act": "gelu",
         "train": False},
        # one window of the language model in training, 32-bit throughout
        {"name": "ffn_window", "op": "ffn", "rows": 1120, "dim": 650, "hidden": 2600, "dtype": "fp32", "act": "silu",
         "train": True},
        # a large training batch in bf16
        {"name": "ffn_large", "op": "ffn", "rows": 8192, "dim": 2048, "hidden": 8192, "dtype": "bf16", "act": "silu",
         "train": True},
        # odd sizes everywhere (no row starts on a 16-byte boundary)
        {"name": "ffn_odd", "op": "ffn", "rows": 777, "dim": 1111, "hidden": 2777, "dtype": "fp16", "act": "gelu",
         "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("ln", "drop", "ffn"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    train = rng.random() < 0.7
    if op == "ffn":
        most = 8192 * 2048 * 8192 // (6 if dtype == "fp32" else 1)
        while True:
            rows, dim, hidden = _log_int(rng, 1, 16384), _log_int(rng, 32, 4096), _log_int(rng, 32, 16384)
            if rng.random() < 0.5:      # half of the models have widths that are multiples of eight
                dim, hidden = (dim + 7) // 8 * 8, (hidden + 7) // 8 * 8
            if rows * dim * hidden <= most:
                break
        return {"op": op, "rows": rows, "dim": dim, "hidden": hidden, "dtype": dtype,
                "act": rng.choice(("silu", "gelu", "relu", "sigmoid")), "train": train}
    most = 16384 * 4096 // (2 if dtype == "fp32" else 1)
    while True:
        rows, dim = _log_int(rng, 1, 65536), _log_int(rng, 2, 16384)
        if rng.random() < 0.5:
            dim = (dim + 7) // 8 * 8
        if rows * dim <= most:
            break
    if op == "ln":
        return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "wide_w": rng.random() < 0.5, "train": train}
    return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "p": round(rng.uniform(0.02, 0.7), 2),
            "site": rng.randrange(64), "residual": rng.random() < 0.5, "train": train}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, rows, dim = DTYPES[case["dtype"]], case["rows"], case["dim"]

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return torch.randn(*shape, device="cuda", generator=g).mul_(scale).add_(shift).to(dtype)

    s = {"case": case}
    train = case["train"]
    if case["op"] == "ln":
        # a residual stream: rows of different scale and offset
        scale = torch.rand(rows, 1, device="cuda", generator=g).mul_(3).add_(0.3)
        shift = torch.randn(rows, 1, device="cuda", generator=g)
        s["x"] = (torch.randn(rows, dim, device="cuda", generator=g) * scale + shift).to(dt).requires_grad_(train)
        wd = torch.float32 if case["wide_w"] else dt
        s["w"] = normal(dim, scale=0.2, shift=1.0, dtype=wd).requires_grad_(train)
        s["b"] = normal(dim, scale=0.2, dtype=wd).requires_grad_(train)
        s["dy"] = normal(rows, dim) if train else None
    elif case["op"] == "drop":
        s["x"] = normal(rows, dim).requires_grad_(train)
        s["r"] = normal(rows, dim, scale=2.0) if case["residual"] else None
        s["key"] = torch.randint(-(1 << 63), (1 << 63) - 1, (1,), device="cuda", generator=g)
        s["dy"] = normal(rows, dim) if train else None
    else:
        hidden = case["hidden"]
        s["x"] = normal(rows, dim).requires_grad_(train)
        s["w_in"] = normal(2 * hidden, dim, scale=dim ** -0.5).requires_grad_(train)
        s["w_out"] = normal(dim, hidden, scale=hidden ** -0.5).requires_grad_(train)
        s["dy"] = normal(rows, dim) if train else None
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    with torch.no_grad():
        return {"ln": _ln, "drop": _drop, "ffn": _ffn}[case["op"]](case, state)


def _own(case, s):
    if case["op"] == "ln":
        from chocosgd_b200.ops.norm import layer_norm

        y = layer_norm(s["x"], s["w"], s["b"], EPS)
        leaves = (s["x"], s["w"], s["b"])
    elif case["op"] == "drop":
        from chocosgd_b200.ops.dropout import dropout

        y = dropout(s["x"], case["p"], s["key"], site=case["site"], residual=s["r"])
        leaves = (s["x"],)
    else:
        from chocosgd_b200.ops.ffn import gated_ffn

        y = gated_ffn(s["x"], s["w_in"], s["w_out"], act=case["act"])
        leaves = (s["x"], s["w_in"], s["w_out"])
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


def _ln(case, s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    xc = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xh = xc * rstd
    y = (xh * w + b).to(s["x"].dtype)
    if not case["train"]:
        return [y]
    dy = s["dy"].float()
    g = dy * w
    dx = (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)) * rstd
    return [y, dx.to(s["x"].dtype), (dy * xh).sum(0).to(s["w"].dtype), dy.sum(0).to(s["b"].dtype)]


def _mulhilo(m, c):
    """High and low word of the 64-bit product of two 32-bit words, in signed 64-bit integers."""
    a, b = m * (c >> 16), m * (c & 0xFFFF)            # both below 2^48
    mid = (a & 0xFFFF) * 65536 + b                    # below 2^32 + 2^48
    return (a >> 16) + (mid >> 32), mid & MASK


def _draws(n, key, site):
    """The 16-bit draws of elements 0 .. n - 1: eight per counter (i / 8 low, i / 8 high, site, 0), ten rounds, the low
    half of a word before its high half."""
    i = torch.arange((n + 7) // 8, device=key.device)
    c0, c1 = i & MASK, i >> 32
    c2, c3 = torch.full_like(i, site), torch.zeros_like(i)
    k0, k1 = key & MASK, (key >> 32) & MASK
    for _ in range(10):
        h0, l0 = _mulhilo(M0, c0)
        h1, l1 = _mulhilo(M1, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + W0) & MASK, (k1 + W1) & MASK
    words = torch.stack((c0, c1, c2, c3), 1)
    return torch.stack((words & 0xFFFF, words >> 16), 2).view(-1)[:n]


def _drop(case, s):
    x, p = s["x"], case["p"]
    drop = int(round(p * 65536))                      # the probability in steps of 2^-16
    keep = (_draws(x.numel(), s["key"], case["site"]) >= drop).view_as(x)
    scale = 65536 / (65536 - drop)
    y = torch.where(keep, x.float() * scale, 0.0)
    y = (y if s["r"] is None else y + s["r"].float()).to(x.dtype)
    if not case["train"]:
        return [y]
    return [y, torch.where(keep, s["dy"].float() * scale, 0.0).to(x.dtype)]


def _act(name, z):
    """The activation and its derivative."""
    if name == "silu":
        sg = torch.sigmoid(z)
        return z * sg, sg * (1 + z * (1 - sg))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "relu":
        return torch.clamp(z, min=0), (z > 0).to(z.dtype)
    sg = torch.sigmoid(z)
    return sg, sg * (1 - sg)


def _ffn(case, s):
    dt, f = s["x"].dtype, case["hidden"]
    x, w_in, w_out = s["x"].float(), s["w_in"].float(), s["w_out"].float()
    z = x @ w_in.t()
    gate, up = z[:, :f], z[:, f:]
    a, da = _act(case["act"], gate)
    h = a * up
    y = (h @ w_out.t()).to(dt)
    if not case["train"]:
        return [y]
    dy = s["dy"].float()
    dh = dy @ w_out
    dz = torch.cat((dh * up * da, dh * a), 1)
    return [y, (dz @ w_in).to(dt), (dz.t() @ x).to(dt), (dy.t() @ h).to(dt)]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    n, dim, train = case["rows"] * case["dim"], case["dim"], case["train"]
    if case["op"] == "ln":
        we = 4 if case["wide_w"] else e
        if not train:
            return {"bytes": 2 * n * e + 2 * dim * we, "flops": 8 * n}
        # x, dy in; y, dx out; the parameters in, their gradients out
        return {"bytes": 4 * n * e + 4 * dim * we, "flops": 22 * n}
    if case["op"] == "drop":
        streams = 2 + int(case["residual"]) + (2 if train else 0)
        return {"bytes": streams * n * e + 8, "flops": (2 if train else 1) * 2 * n}
    wts = 3 * dim * case["hidden"]
    flops = 2 * case["rows"] * wts
    if not train:
        return {"bytes": (2 * n + wts) * e, "flops": flops}
    return {"bytes": (4 * n + 2 * wts) * e, "flops": 3 * flops}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "ln":
            return _exact_ln(case, s)
        if case["op"] == "drop":
            return _exact_drop(case, s)
        return _exact_ffn(case, s)


def _exact_ln(case, s):
    x, w, b = (s[k].double() for k in ("x", "w", "b"))
    d = x.shape[1]
    mu = x.sum(1) / d
    var = ((x - mu[:, None]) ** 2).sum(1) / d
    sigma = torch.sqrt(var + EPS)
    z = (x - mu[:, None]) / sigma[:, None]
    y = torch.addcmul(b, z, w)
    if not case["train"]:
        return [y]
    dy = s["dy"].double()
    dz = dy * w
    # d z_j / d x_i = (delta_ij - 1/d - z_i z_j / d) / sigma
    along_z = torch.einsum("ij,ij->i", dz, z) / d
    dx = (dz - (dz.sum(1) / d)[:, None] - z * along_z[:, None]) / sigma[:, None]
    return [y, dx, torch.einsum("ij,ij->j", dy, z), dy.sum(0)]


def _exact_drop(case, s):
    n = s["x"].numel()
    if n > 1 << 26:
        return None
    k = int(s["key"].item()) & ((1 << 64) - 1)
    k0, k1 = k & MASK, k >> 32
    low = np.uint64(MASK)
    i = np.arange((n + 7) // 8, dtype=np.uint64)
    c = [i & low, i >> np.uint64(32), np.full_like(i, case["site"]), np.zeros_like(i)]
    for r in range(10):
        p0, p1 = c[0] * np.uint64(M0), c[2] * np.uint64(M1)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64((k0 + r * W0) & MASK), p1 & low,
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64((k1 + r * W1) & MASK), p0 & low]
    u = np.stack(c, 1).astype("<u4").view("<u2").reshape(-1)[:n]
    q = round(case["p"] * 2.0 ** 16) / 2.0 ** 16
    kept = torch.from_numpy(u / 2.0 ** 16 >= q).to(s["x"].device).view(s["x"].shape)
    m = kept.double() / (1.0 - q)
    y = s["x"].double() * m
    if s["r"] is not None:
        y = y + s["r"].double()
    return [y, s["dy"].double() * m] if case["train"] else [y]


def _exact_ffn(case, s):
    f = case["hidden"]
    x, wo = s["x"].double(), s["w_out"].double()
    wg, wu = s["w_in"][:f].double(), s["w_in"][f:].double()
    g, u = torch.einsum("md,fd->mf", x, wg), torch.einsum("md,fd->mf", x, wu)
    kind = case["act"]
    if kind == "gelu":
        cdf = torch.special.ndtr(g)
        a, slope = g * cdf, cdf + g * torch.exp(-g * g / 2) / (2 * math.pi) ** 0.5
    elif kind == "relu":
        a, slope = torch.relu(g), torch.heaviside(g, torch.zeros((), dtype=g.dtype, device=g.device))
    else:
        sg = 1 / (1 + torch.exp(-g))
        a, slope = (sg, sg - sg * sg) if kind == "sigmoid" else (g * sg, sg + g * sg - g * sg * sg)
    h = a * u
    y = torch.einsum("mf,nf->mn", h, wo)
    if not case["train"]:
        return [y]
    dy = s["dy"].double()
    dwo = torch.einsum("mn,mf->nf", dy, h)
    dh = torch.einsum("mn,nf->mf", dy, wo)
    dg, du = dh * u * slope, dh * a
    dx = torch.einsum("mf,fd->md", dg, wg) + torch.einsum("mf,fd->md", du, wu)
    dwi = torch.cat((torch.einsum("mf,md->fd", dg, x), torch.einsum("mf,md->fd", du, x)), 0)
    return [y, dx, dwi, dwo]
