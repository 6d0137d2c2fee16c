"""Measured cases of the per-voxel gated feed-forward block and of the fused
residual norms around it, forward and backward.

``run`` computes a case either in its plain form (elementary torch operations
in 32 bits, rounded once at the end) or, where ``own`` is true, through the
executor of this package.  Rows are voxels of a level (or one global token),
``[n, c]`` row-major as everywhere in this package; a row's sample index is
field 3 of its coordinates.

    gated_ffn          y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd
    gated_ffn_backward the gradients of x, the weights and the biases; the
                       hidden values are computed again from x
    residual_norm      r = s x + gate * Norm_post(f);  h = Norm_pre(r)
    residual_norm_backward  the gradients of x, f, the gate and the norms'
                       weights from the gradients of r and h
"""

import math
import random

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6
_executor = None


def _ex():
    global _executor
    if _executor is None:
        from mogecpp_b200.sparse import SparseCudaExecutor
        _executor = SparseCudaExecutor(torch.cuda.current_device())
    return _executor


# ------------------------------------------------------------------ cases
def _ffn(name, op, n, c, hidden, dtype, act, bias):
    return {"name": name, "op": op, "n": n, "c": c, "hidden": hidden, "dtype": dtype, "act": act, "bias": bias}


def _norm(name, op, n, c, x_dtype, f_dtype, post, pre, gate, nsamples, res_scale):
    return {"name": name, "op": op, "n": n, "c": c, "x_dtype": x_dtype, "f_dtype": f_dtype, "post": post,
            "pre": pre, "gate": gate, "nsamples": nsamples, "res_scale": res_scale}


def listed():
    return [
        # one global token through a wide block: the weights are read once, latency counts
        _ffn("ffn_one_token", "ffn", 1, 1024, 4096, "bf16", "silu", False),
        # the coarsest level of a small image: few rows, hidden size no multiple of a tile
        _ffn("ffn_coarse_level", "ffn", 1237, 512, 1376, "f16", "gelu", True),
        # every voxel of a 128^3 level at 64 channels
        _ffn("ffn_level_c64", "ffn", 101117, 64, 256, "f16", "gelu_erf", True),
        # every voxel of a 256^3 level at 128 channels
        _ffn("ffn_level_c128", "ffn", 402131, 128, 512, "bf16", "silu", False),
        # tokens of a batch of images through a wide block
        _ffn("ffn_wide", "ffn", 8192, 1024, 4096, "bf16", "silu", True),
        # training step of a coarse level, ragged hidden size
        _ffn("ffn_bwd_coarse_level", "ffn_bwd", 1237, 256, 680, "f16", "gelu", True),
        # training step of a fine level: few channels, sums over many rows
        _ffn("ffn_bwd_level_c128", "ffn_bwd", 101117, 128, 512, "bf16", "silu", True),
        # training step of a wide block
        _ffn("ffn_bwd_wide", "ffn_bwd", 8192, 1024, 4096, "bf16", "silu", False),
        # one global token between two blocks: latency
        _norm("norm_one_token", "norm", 1, 1024, "bf16", "bf16", "rms", "rms", "channel", 1, 1.0),
        # every voxel of a 256^3 level, two samples with a gate each
        _norm("norm_level_c128", "norm", 402131, 128, "bf16", "bf16", "layer", "layer", "sample", 2, 1.0),
        # coarse level, 32-bit residual stream with 16-bit branches
        _norm("norm_bwd_coarse_level", "norm_bwd", 1237, 512, "f32", "f16", "rms", "layer", "channel", 1, 0.7),
        # training step at every voxel of a 256^3 level
        _norm("norm_bwd_level_c128", "norm_bwd", 402131, 128, "bf16", "bf16", "layer", "rms", "sample", 2, 1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["ffn", "ffn_bwd", "norm", "norm_bwd"])
    c = 8 * _log_int(rng, 8, 128)
    n = _log_int(rng, 1, 400000)
    if op in ("ffn", "ffn_bwd"):
        hidden = 8 * max(1, int(round(c * rng.uniform(1.5, 4.0) / 8)))
        cap = 2.5e10 if op == "ffn" else 1.2e10   # rows * channels * hidden
        n = max(1, min(n, int(cap / (c * hidden))))
        return {"op": op, "n": n, "c": c, "hidden": hidden, "dtype": rng.choice(["bf16", "f16"]),
                "act": rng.choice(["silu", "gelu", "gelu_erf"]), "bias": rng.random() < 0.5}
    n = max(1, min(n, int(4e7 / c)))
    gate = rng.choice(["none", "channel", "sample"])
    f_dtype = rng.choice(["bf16", "f16"])
    kinds = ["layer", "rms"]
    return {"op": op, "n": n, "c": c, "x_dtype": rng.choice(["f32", f_dtype]), "f_dtype": f_dtype,
            "post": rng.choice(kinds + ["none"]), "pre": rng.choice(kinds), "gate": gate,
            "nsamples": rng.randint(2, 9) if gate == "sample" else 1, "res_scale": rng.choice([1.0, 0.7])}


# ----------------------------------------------------------------- inputs
def _randn(gen, shape, scale=1.0, shift=0.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale + shift


def _sample_of_row(case, gen):
    """Rows sorted by sample, samples of unequal size."""
    cuts = torch.rand(case["nsamples"] - 1, generator=gen, device="cuda").sort().values * case["n"]
    rows = torch.arange(case["n"], device="cuda")
    return (rows[:, None] >= cuts[None, :]).sum(1) if case["nsamples"] > 1 else torch.zeros_like(rows)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n, c = case["n"], case["c"]
    st = {"case": case}
    if own:
        st["ex"] = _ex()
    if case["op"] in ("ffn", "ffn_bwd"):
        dt, hd = _DT[case["dtype"]], case["hidden"]
        # x comes out of a norm with a learned weight: unit rows, channels of unequal scale
        st["x"] = (_randn(gen, (n, c)) * _randn(gen, (c,), 0.2, 1.0)).to(dt)
        ffn = {"w_gate": _randn(gen, (hd, c), c ** -0.5).to(dt), "w_up": _randn(gen, (hd, c), c ** -0.5).to(dt),
               "w_down": _randn(gen, (c, hd), hd ** -0.5).to(dt)}
        if case["bias"]:
            ffn["b_gate"] = _randn(gen, (hd,), 0.1)
            ffn["b_up"] = _randn(gen, (hd,), 0.1)
            ffn["b_down"] = _randn(gen, (c,), 0.1)
        st["ffn"] = ffn
        if case["op"] == "ffn_bwd":
            st["dy"] = _randn(gen, (n, c), 0.1).to(dt)
        return st
    xd, fd = _DT[case["x_dtype"]], _DT[case["f_dtype"]]
    mean = _randn(gen, (c,), 0.5)
    st["x"] = (_randn(gen, (n, c), 1.5) + mean).to(xd)   # the residual stream (r where gradients are asked for)
    st["f"] = (_randn(gen, (n, c), 0.8) + 0.3 * mean).to(fd)
    for which in ("post", "pre"):
        kind = case[which]
        st[which] = None
        if kind != "none":
            st[which] = {"kind": kind, "w": _randn(gen, (c,), 0.1, 1.0), "eps": _EPS,
                         "b": _randn(gen, (c,), 0.1) if kind == "layer" else None}
    st["gate"] = st["coords"] = None
    if case["gate"] == "channel":
        st["gate"] = _randn(gen, (c,), 0.2, 0.4)
    elif case["gate"] == "sample":
        st["gate"] = _randn(gen, (case["nsamples"], c), 0.2, 0.4)
        st["coords"] = torch.randint(0, 256, (n, 4), generator=gen, device="cuda", dtype=torch.int32)
        st["coords"][:, 3] = _sample_of_row(case, gen).to(torch.int32)
    if case["op"] == "norm_bwd":
        st["dy"] = _randn(gen, (n, c), 0.1).to(xd)
        st["dh"] = _randn(gen, (n, c), 0.1).to(fd)
    return st


# ------------------------------------------------------------ plain forms
_K0 = math.sqrt(2.0 / math.pi)
_K1 = 0.044715


def _act32(g, act):
    """Activation and its derivative."""
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if act == "gelu":
        t = torch.tanh(_K0 * (g + _K1 * g * g * g))
        return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * _K0 * (1.0 + 3.0 * _K1 * g * g)
    p = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * p, p + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _hidden32(st):
    x, w = st["x"].float(), st["ffn"]
    g = torch.matmul(x, w["w_gate"].float().t())
    u = torch.matmul(x, w["w_up"].float().t())
    if "b_gate" in w:
        g, u = g + w["b_gate"], u + w["b_up"]
    return x, g, u


def _plain_ffn(st):
    case, w = st["case"], st["ffn"]
    _, g, u = _hidden32(st)
    y = torch.matmul(_act32(g, case["act"])[0] * u, w["w_down"].float().t())
    if "b_down" in w:
        y = y + w["b_down"]
    return y.to(st["x"].dtype)


def _plain_ffn_bwd(st):
    case, w, dt = st["case"], st["ffn"], st["x"].dtype
    x, g, u = _hidden32(st)
    a, da = _act32(g, case["act"])
    dy = st["dy"].float()
    dh = torch.matmul(dy, w["w_down"].float())
    dg, du = dh * u * da, dh * a
    out = [(torch.matmul(dg, w["w_gate"].float()) + torch.matmul(du, w["w_up"].float())).to(dt),
           torch.matmul(dg.t(), x).to(dt), torch.matmul(du.t(), x).to(dt), torch.matmul(dy.t(), a * u).to(dt)]
    if "b_gate" in w:
        out += [t.sum(0, dtype=torch.float64).float() for t in (dg, du, dy)]
    return out


def _norm32(v, nrm):
    """Normalised rows and 1 / their scale."""
    if nrm["kind"] == "layer":
        v = v - v.mean(1, keepdim=True)
    rs = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + nrm["eps"])
    return v * rs, rs


def _affine32(v, nrm):
    v = v * nrm["w"]
    return v if nrm["b"] is None else v + nrm["b"]


def _gate32(st):
    if st["gate"] is None:
        return None
    return st["gate"] if st["coords"] is None else st["gate"][st["coords"][:, 3].long()]


def _plain_norm(st):
    t = st["f"].float()
    if st["post"] is not None:
        t = _affine32(_norm32(t, st["post"])[0], st["post"])
    gate = _gate32(st)
    r = st["case"]["res_scale"] * st["x"].float() + (t if gate is None else gate * t)
    h = _affine32(_norm32(r, st["pre"])[0], st["pre"])
    return r.to(st["x"].dtype), h.to(st["f"].dtype)


def _norm_back32(dn, v_hat, rs, nrm):
    d = dn * nrm["w"]
    if nrm["kind"] == "layer":
        d = d - d.mean(1, keepdim=True)
    return rs * (d - v_hat * (d * v_hat).mean(1, keepdim=True))


def _plain_norm_bwd(st):
    case = st["case"]
    r, f, dy, dh = st["x"].float(), st["f"].float(), st["dy"].float(), st["dh"].float()
    pre, post, gate = st["pre"], st["post"], _gate32(st)
    r_hat, r_rs = _norm32(r, pre)
    dr = dy + _norm_back32(dh, r_hat, r_rs, pre)
    t, f_hat, f_rs = f, None, None
    if post is not None:
        f_hat, f_rs = _norm32(f, post)
        t = _affine32(f_hat, post)
    dt = dr if gate is None else gate * dr
    df = dt if post is None else _norm_back32(dt, f_hat, f_rs, post)
    out = [(case["res_scale"] * dr).to(st["x"].dtype), df.to(st["f"].dtype)]

    def cols(v):
        return v.sum(0, dtype=torch.float64).float()
    if case["gate"] == "channel":
        out.append(cols(dr * t))
    elif case["gate"] == "sample":
        sample = st["coords"][:, 3]
        out.append(torch.stack([cols((dr * t)[sample == s]) for s in range(case["nsamples"])]))
    if post is not None:
        out.append(cols(dt * f_hat))
        if post["b"] is not None:
            out.append(cols(dt))
    out.append(cols(dh * r_hat))
    if pre["b"] is not None:
        out.append(cols(dh))
    return out


# -------------------------------------------------------------------- run
def run(st):
    case = st["case"]
    if not own:
        return {"ffn": _plain_ffn, "ffn_bwd": _plain_ffn_bwd, "norm": _plain_norm,
                "norm_bwd": _plain_norm_bwd}[case["op"]](st)
    ex = st["ex"]
    if case["op"] == "ffn":
        return ex.gated_ffn(st["x"], st["ffn"], act=case["act"])
    if case["op"] == "ffn_bwd":
        g = ex.gated_ffn_backward(st["x"], st["dy"], st["ffn"], act=case["act"])
        keys = ["x", "w_gate", "w_up", "w_down"] + (["b_gate", "b_up", "b_down"] if case["bias"] else [])
        return [g[k] for k in keys]
    cfg = dict(post=st["post"], gate=st["gate"], pre=st["pre"], res_scale=case["res_scale"], coords=st["coords"])
    if case["op"] == "norm":
        return ex.residual_norm(st["x"], st["f"], **cfg)
    g = ex.residual_norm_backward(st["x"], st["f"], st["dy"], st["dh"], **cfg)
    return [g[k] for k in ("x", "f", "gate", "post_w", "post_b", "pre_w", "pre_b") if g.get(k) is not None]


# ------------------------------------------------------------------ exact
def _act64(g, act):
    if act == "silu":
        return g * torch.sigmoid(g)
    if act == "gelu":
        return g * torch.sigmoid(2.0 * _K0 * (g + _K1 * g ** 3))
    return g * 0.5 * torch.erfc(-g / math.sqrt(2.0))


def _norm64(v, kind, w, b, eps):
    if kind == "layer":
        var, mean = torch.var_mean(v, dim=1, correction=0, keepdim=True)
        out = (v - mean) / torch.sqrt(var + eps) * w
    else:
        out = v / torch.sqrt(v.square().mean(1, keepdim=True) + eps) * w
    return out if b is None else out + b


def exact(case, seed):
    st = prepare(case, seed)

    def leaf(t):
        return None if t is None else t.double().requires_grad_(case["op"].endswith("_bwd"))
    if case["op"] in ("ffn", "ffn_bwd"):
        x = leaf(st["x"])
        p = {k: leaf(v) for k, v in st["ffn"].items()}

        def block(xs):
            g, u = xs @ p["w_gate"].mT, xs @ p["w_up"].mT
            if case["bias"]:
                g, u = g + p["b_gate"], u + p["b_up"]
            y = (_act64(g, case["act"]) * u) @ p["w_down"].mT
            return y + p["b_down"] if case["bias"] else y
        if case["op"] == "ffn":
            return torch.cat([block(xs) for xs in x.split(65536)])
        for i in range(0, case["n"], 65536):
            (block(x[i:i + 65536]) * st["dy"][i:i + 65536].double()).sum().backward()
        keys = ["w_gate", "w_up", "w_down"] + (["b_gate", "b_up", "b_down"] if case["bias"] else [])
        return [x.grad] + [p[k].grad for k in keys]
    x, f, gate = leaf(st["x"]), leaf(st["f"]), leaf(st["gate"])
    w = {(k, q): leaf(st[k][q]) for k in ("post", "pre") if st[k] is not None for q in ("w", "b")}

    def pre(r):
        return _norm64(r, case["pre"], w["pre", "w"], w["pre", "b"], _EPS)

    def branch():
        t = f if case["post"] == "none" else _norm64(f, case["post"], w["post", "w"], w["post", "b"], _EPS)
        if gate is None:
            return t
        return t * (gate if st["coords"] is None else gate.index_select(0, st["coords"][:, 3].long()))
    if case["op"] == "norm":
        r = case["res_scale"] * x + branch()
        return r, pre(r)
    (pre(x) * st["dh"].double()).sum().backward()
    dr = x.grad + st["dy"].double()
    (branch() * dr).sum().backward()
    out = [case["res_scale"] * dr, f.grad] + ([] if gate is None else [gate.grad])
    for k in (("post", "w"), ("post", "b"), ("pre", "w"), ("pre", "b")):
        if w.get(k) is not None:
            out.append(w[k].grad)
    return out


# ------------------------------------------------------------------- work
def work(case):
    """Bytes: inputs once, outputs once.  Flops: the products (the backward
    pass of the block computes its two hidden projections again); for the
    norms some ten operations an element each way."""
    n, c = case["n"], case["c"]
    if case["op"] in ("ffn", "ffn_bwd"):
        hd = case["hidden"]
        weights = 3 * c * hd * 2
        bias = (2 * hd + c) * 4 if case["bias"] else 0
        if case["op"] == "ffn":
            return {"bytes": 2 * n * c * 2 + weights + bias, "flops": 6 * n * c * hd}
        return {"bytes": 3 * n * c * 2 + 2 * weights + 2 * bias, "flops": 16 * n * c * hd}
    xb, fb = (4 if case["x_dtype"] == "f32" else 2), (4 if case["f_dtype"] == "f32" else 2)
    coords = 16 * n if case["gate"] == "sample" else 0
    small = 4 * c * (4 + case["nsamples"])
    if case["op"] == "norm":
        return {"bytes": n * c * (2 * xb + 2 * fb) + coords + small, "flops": 16 * n * c}
    return {"bytes": n * c * (3 * xb + 3 * fb) + coords + 2 * small, "flops": 40 * n * c}
