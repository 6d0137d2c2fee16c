"""Gated feed-forward block, forward and backward, and the stack of residual
feed-forward blocks, against plain 64-bit formulas.

Tolerances.  A value stored in 16 bits is off by at most u = eps / 2 of itself.
The hidden values (and dg, du) are rounded once to the features' type before
the second product, and the output once more.  For y = sum_j h_j w_j the first
rounding contributes at most u sum_j |h_j w_j|, the second u |y|, and the
tensor core's fp32 sums at most (K + 16) 2^-23 of the absolute sum (each of K
additions truncated, 16 for the activation's approximations).  So an element
is within u |y| + (u + (K + 16) 2^-23) A of its exact value, A the same sum
over absolute values, plus half the smallest subnormal of fp16 (2^-25) per
rounded value.  The hidden values' own error, from the fp32 sums over c and
the activation (relative slope at most ~1 + |g|), enters A with the factor
(c + 16) 2^-23 (1 + max|g|)."""
import math

import pytest
import torch

from mogecpp_b200.lib import MscError

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -25


def act64(g, act):
    """Activation and derivative."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)
    p = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def make(seed, n, c, hidden, dtype, bias, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape, s=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * s
    ffn = dict(w_gate=r(hidden, c, s=c ** -0.5).to(dtype), w_up=r(hidden, c, s=c ** -0.5).to(dtype),
               w_down=r(c, hidden, s=hidden ** -0.5).to(dtype))
    if bias:
        ffn.update(b_gate=r(hidden, s=0.2), b_up=r(hidden, s=0.2), b_down=r(c, s=0.2))
    return (r(n, c) * scale).to(dtype), r(n, c, s=0.3).to(dtype), ffn


def parts(x, ffn, act):
    x = x.double()
    w = {k: v.double() for k, v in ffn.items()}
    g, u = x @ w["w_gate"].T, x @ w["w_up"].T
    if "b_gate" in w:
        g, u = g + w["b_gate"], u + w["b_up"]
    return x, w, g, u, *act64(g, act)


def fwd_bound(x, ffn, act, dtype):
    x, w, g, u, a, _ = parts(x, ffn, act)
    h = a * u
    y = h @ w["w_down"].T + w.get("b_down", 0.0)
    us = torch.finfo(dtype).eps / 2
    hidden, c = ffn["w_gate"].shape
    # an absolute sum that also covers the cancellation inside g and u
    au = x.abs() @ w["w_up"].abs().T + w["b_up"].abs() if "b_up" in w else x.abs() @ w["w_up"].abs().T
    ag = x.abs() @ w["w_gate"].abs().T + w["b_gate"].abs() if "b_gate" in w else x.abs() @ w["w_gate"].abs().T
    f32 = 2.0 ** -23
    dh = (c + 16) * f32 * (a.abs() * au + 1.2 * ag * u.abs()) + 16 * f32 * h.abs()
    big = (h.abs() * (us + (hidden + 16) * f32) + dh + TINY) @ w["w_down"].abs().T
    return y, us * y.abs() + (1 + us) * big + TINY + 4 * f32 * y.abs()


def check(got, want, bound, what):
    err = (got.double() - want).abs()
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert got.isfinite().all(), what
    assert worst <= 1.0, f"{what}: {worst} of the bound"


# lengths of one, below and above a tile, channels and hidden sizes that end inside a tile of 64 / 128 / 256,
# few rows (dot products, K split), many (one kernel up to 128 channels, CTA pairs)
SHAPES = [(1, 64, 64), (1, 1024, 2048), (3, 8, 8), (8, 128, 512), (9, 128, 520), (127, 64, 256), (128, 128, 512),
          (129, 136, 344), (300, 264, 72), (1237, 512, 1376), (5000, 72, 200), (20000, 128, 512), (20001, 64, 176),
          (2000, 1024, 1032), (19001, 8, 8), (19201, 120, 72), (10007, 264, 520), (4097, 1024, 2056)]


@pytest.mark.parametrize("n,c,hidden", SHAPES)
@pytest.mark.parametrize("dtype,act,bias", [(torch.bfloat16, "silu", True), (torch.float16, "gelu", False),
                                            (torch.float16, "gelu_erf", True)])
def test_forward(ex, n, c, hidden, dtype, act, bias):
    x, _, ffn = make(n + c, n, c, hidden, dtype, bias)
    y = ex.gated_ffn(x, ffn, act=act)
    ex.check()
    want, bound = fwd_bound(x, ffn, act, dtype)
    check(y, want, bound, "y")


def bwd_reference(x, dy, ffn, act, dtype):
    """Exact gradients and their bounds (see the module's derivation; the
    rounded operands are dg, du and h, with the fp32 error of each)."""
    x, w, g, u, a, da = parts(x, ffn, act)
    dy = dy.double()
    us, f32 = torch.finfo(dtype).eps / 2, 2.0 ** -23
    hidden, c = ffn["w_gate"].shape
    n = x.shape[0]
    dh = dy @ w["w_down"]
    dg, du, h = dh * u * da, dh * a, a * u
    ax = x.abs()
    eu = (c + 16) * f32 * (ax @ w["w_up"].abs().T + (w["b_up"].abs() if "b_up" in w else 0))
    eg = (c + 16) * f32 * (ax @ w["w_gate"].abs().T + (w["b_gate"].abs() if "b_gate" in w else 0))
    ed = (c + 16) * f32 * (dy.abs() @ w["w_down"].abs())
    # |act'| <= 1.2, |act''| <= 0.8
    e_dg = (ed * u * da).abs() + (dh * eu * da).abs() + 0.8 * (dh * u).abs() * eg + 16 * f32 * (dh * u).abs() * 1.2
    e_du = (ed * a).abs() + 1.2 * dh.abs() * eg + 16 * f32 * du.abs()
    e_h = 1.2 * eg * u.abs() + a.abs() * eu + 16 * f32 * h.abs()
    r_dg, r_du, r_h = e_dg + us * dg.abs() + TINY, e_du + us * du.abs() + TINY, e_h + us * h.abs() + TINY
    out, bnd = {}, {}

    def put(k, want, operand, chain, absum):
        out[k] = want
        bnd[k] = (1 + us) * (operand + (chain + 16) * f32 * absum) + us * want.abs() + TINY
    put("x", dg @ w["w_gate"] + du @ w["w_up"], r_dg @ w["w_gate"].abs() + r_du @ w["w_up"].abs(), 2 * hidden,
        dg.abs() @ w["w_gate"].abs() + du.abs() @ w["w_up"].abs())
    put("w_gate", dg.T @ x, r_dg.T @ ax, n, dg.abs().T @ ax)
    put("w_up", du.T @ x, r_du.T @ ax, n, du.abs().T @ ax)
    put("w_down", dy.T @ h, dy.abs().T @ r_h, n, dy.abs().T @ h.abs())
    # the bias sums use the unrounded values: fp32 sums of 128 rows, then double
    for k, v, e in (("b_gate", dg, e_dg), ("b_up", du, e_du)):
        out[k] = v.sum(0)
        bnd[k] = e.sum(0) + 140 * f32 * v.abs().sum(0) + f32 * out[k].abs() + 1e-30
    out["b_down"] = dy.sum(0)
    bnd["b_down"] = 260 * f32 * dy.abs().sum(0) + f32 * out["b_down"].abs() + 1e-30
    return out, bnd


@pytest.mark.parametrize("n,c,hidden", SHAPES)
@pytest.mark.parametrize("dtype,act,bias", [(torch.bfloat16, "silu", True), (torch.float16, "gelu", True),
                                            (torch.bfloat16, "gelu_erf", False)])
def test_backward(ex, n, c, hidden, dtype, act, bias):
    x, dy, ffn = make(2 * n + c, n, c, hidden, dtype, bias)
    got = ex.gated_ffn_backward(x, dy, ffn, act=act)
    ex.check()
    want, bound = bwd_reference(x, dy, ffn, act, dtype)
    assert set(got) == {"x"} | set(ffn)
    for k in got:
        check(got[k], want[k], bound[k], k)
    only_x = ex.gated_ffn_backward(x, dy, ffn, act=act, weights=False)
    assert set(only_x) == {"x"} and torch.equal(only_x["x"], got["x"])


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_erf"])
def test_gradient_against_differences(ex, act):
    """Directional derivatives of the 64-bit block along one direction of each
    input, by central differences.  Step 1e-4 of a smooth function with third
    derivatives of order one: error ~1e-8 of the scale; the kernel's gradients
    carry u = 2^-11 twice per product (3 u of the absolute sums covers both)."""
    x, dy, ffn = make(7, 150, 72, 136, torch.float16, True)
    got = ex.gated_ffn_backward(x, dy, ffn, act=act)
    _, bound = bwd_reference(x, dy, ffn, act, torch.float16)

    def loss(xx, p):
        g, u = xx @ p["w_gate"].T + p["b_gate"], xx @ p["w_up"].T + p["b_up"]
        return ((act64(g, act)[0] * u @ p["w_down"].T + p["b_down"]) * dy.double()).sum().item()
    p = {k: v.double() for k, v in ffn.items()}
    gen = torch.Generator(device="cuda").manual_seed(8)
    for k in got:
        base = x.double() if k == "x" else p[k]
        d = torch.randn(base.shape, generator=gen, device="cuda", dtype=torch.float64)
        d /= d.norm()
        eps = 1e-4

        def at(s):
            v = base + s * d
            return loss(v, p) if k == "x" else loss(x.double(), {**p, k: v})
        diff = (at(eps) - at(-eps)) / (2 * eps)
        along = (got[k].double() * d).sum().item()
        assert abs(along - diff) <= (bound[k] * d.abs()).sum().item() + 1e-6 * (1 + abs(diff)), k


def test_empty_and_in_place(ex):
    x, dy, ffn = make(9, 200, 128, 256, torch.bfloat16, True)
    e = x[:0].contiguous()
    assert ex.gated_ffn(e, ffn).shape == (0, 128)
    g = ex.gated_ffn_backward(e, e, ffn)
    assert all(not v.any() for v in g.values())   # sums over no rows are zero
    want = ex.gated_ffn(x, ffn)
    y = x.clone()
    ex.gated_ffn(y, ffn, out=y)
    assert torch.equal(y, want)


def test_same_bits_every_time(ex):
    for n, c, hidden in ((1, 1024, 2048), (700, 128, 344), (20001, 64, 176)):
        x, dy, ffn = make(10, n, c, hidden, torch.bfloat16, True)
        y, g = ex.gated_ffn(x, ffn), ex.gated_ffn_backward(x, dy, ffn)
        for _ in range(3):
            assert torch.equal(y, ex.gated_ffn(x, ffn))
            h = ex.gated_ffn_backward(x, dy, ffn)
            assert all(torch.equal(g[k], h[k]) for k in g)


def test_rows_do_not_mix(ex):
    """A row that holds infinities and NaN spoils its own output row alone,
    and rows past the last one stay as they were."""
    x, _, ffn = make(11, 260, 128, 344, torch.bfloat16, True)
    want = ex.gated_ffn(x, ffn)
    bad = x.clone()
    bad[37] = float("inf")
    bad[130, 5] = float("nan")
    buf = torch.full((300, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    y = ex.gated_ffn(bad, ffn, out=buf[:260])
    keep = [i for i in range(260) if i not in (37, 130)]
    assert torch.equal(y[keep], want[keep])
    assert not y[130].isfinite().any() and not y[37].isfinite().all()
    assert (buf[260:] == 3.0).all()


def test_large_values_stay_finite(ex):
    """Saturated gates: act(g) is g or 0 far out, with no overflow inside."""
    for act in ("silu", "gelu", "gelu_erf"):
        x, dy, ffn = make(12, 64, 64, 64, torch.bfloat16, False, scale=3000.0)
        y = ex.gated_ffn(x, ffn, act=act)
        want, bound = fwd_bound(x, ffn, act, torch.bfloat16)
        check(y, want, bound, act)
        g = ex.gated_ffn_backward(x, dy, ffn, act=act)
        assert all(v.isfinite().all() for v in g.values())


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_erf"])
def test_far_out_gates(ex, act):
    """Gates of exactly -3e5 ... 3e5 (identity weights, fp32-exact products):
    far below zero the value and the derivative are zero (to |g| 2^-62, the
    floor of sigma), far above g and one; a 16-bit rounding each."""
    c = 16
    g = torch.tensor([-3e5, -1e4, -300., -40., -8., -2., -0.5, 0., 0.5, 2., 8., 40., 300., 1e4, 3e5, 1.],
                     device="cuda").to(torch.bfloat16)
    x = g.repeat(40, 1).contiguous()
    eye = torch.eye(c, device="cuda", dtype=torch.bfloat16)
    ffn = dict(w_gate=eye, w_up=torch.zeros_like(eye), w_down=eye, b_up=torch.ones(c, device="cuda"))
    v, dv = act64(g.double(), act)
    y = ex.gated_ffn(x, ffn, act=act)
    u = 2.0 ** -8
    assert ((y.double() - v).abs() <= 2 * u * v.abs() + 1e-6).all()
    got = ex.gated_ffn_backward(x, torch.ones_like(x), ffn, act=act)
    assert ((got["x"].double() - dv).abs() <= 2 * u * dv.abs() + 1e-6).all()
    ex.check()


@pytest.mark.parametrize("n,c,hidden", [(1, 256, 1032), (6, 128, 344), (20001, 64, 176), (19500, 128, 344),
                                        (10000, 264, 520)])
def test_every_path_captured(ex, n, c, hidden):
    """A first call inside a capture, replayed on new data in the same buffers:
    the two launches of few rows, the single kernel, the CTA pairs."""
    x, dy, ffn = make(70 + n, n, c, hidden, torch.bfloat16, True)
    other = make(71 + n, n, c, hidden, torch.bfloat16, True)[0]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = ex.gated_ffn(x, ffn)
        g = ex.gated_ffn_backward(x, dy, ffn)
    for data in (x.clone(), other):
        x.copy_(data)
        gr.replay()
        assert torch.equal(y, ex.gated_ffn(data, ffn))
        want = ex.gated_ffn_backward(data, dy, ffn)
        assert all(torch.equal(g[k], want[k]) for k in want)
    ex.check()


def test_streams_and_graphs(ex):
    """Two streams at once, and two captured graphs replayed in turn, give the
    eager results (every call has its own workspace)."""
    sets = [make(20 + i, 1500, 128, 512, torch.bfloat16, True) for i in range(2)]
    want = [(ex.gated_ffn(x, f), ex.gated_ffn_backward(x, dy, f)) for x, dy, f in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for i, (x, dy, f) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append((ex.gated_ffn(x, f), ex.gated_ffn_backward(x, dy, f)))
    torch.cuda.synchronize()
    for i in range(2):
        for y, g in got[i]:
            assert torch.equal(y, want[i][0]) and all(torch.equal(g[k], want[i][1][k]) for k in g)
    graphs, outs = [], []
    for x, dy, f in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append((ex.gated_ffn(x, f), ex.gated_ffn_backward(x, dy, f)))
        graphs.append(gr)
    for _ in range(3):
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i][0], want[i][0])
            assert all(torch.equal(outs[i][1][k], want[i][1][k]) for k in want[i][1])
    ex.check()


def test_refusals(ex):
    x, dy, ffn = make(30, 16, 64, 128, torch.bfloat16, True)
    with pytest.raises(MscError, match="fp16 and bf16"):
        f32 = {k: v.float() for k, v in ffn.items()}
        ex.gated_ffn(x.float(), f32)
    with pytest.raises(MscError, match="act"):
        ex.gated_ffn(x, ffn, act="relu")
    with pytest.raises(MscError, match="w_up"):
        ex.gated_ffn(x, {**ffn, "w_up": ffn["w_up"][:64].contiguous()})
    with pytest.raises(MscError, match="w_down"):
        ex.gated_ffn(x, {**ffn, "w_down": ffn["w_down"].half()})
    with pytest.raises(MscError, match="contiguous"):
        ex.gated_ffn(x.repeat(1, 2)[:, :64], ffn)
    with pytest.raises(MscError, match="b_gate"):
        ex.gated_ffn(x, {**ffn, "b_gate": ffn["b_gate"].half()})
    with pytest.raises(MscError, match="dy"):
        ex.gated_ffn_backward(x, dy[:8].contiguous(), ffn)
    with pytest.raises(MscError, match="multiples of 8"):
        xx, _, ff = make(31, 4, 60, 128, torch.bfloat16, False)
        ex.gated_ffn(xx, ff)
    with pytest.raises(MscError, match="aligned"):
        flat = torch.zeros(16 * 64 + 1, dtype=torch.bfloat16, device="cuda")
        ex.gated_ffn(flat[1:].view(16, 64), ffn)
    import ctypes as C
    from mogecpp_b200 import lib as L
    f = ex._ffn(ffn, "silu", 64, x.dtype)
    p = C.c_void_p(x.data_ptr())
    g = L.FfnGrads(x.data_ptr(), None, None, None, None, None, None)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    assert ex.lib.msc_gated_ffn(ex.ctx, C.byref(f), 16, 64, p, p, C.c_void_p(ws.data_ptr()), 16, None) == -5
    assert ex.lib.msc_gated_ffn_backward(ex.ctx, C.byref(f), 16, 64, p, C.c_void_p(dy.data_ptr()), C.byref(g),
                                         C.c_void_p(ws.data_ptr()), ws.numel(), None) == -1
    assert b"dx" in ex.lib.msc_last_error()
    part = L.FfnGrads(None, ws.data_ptr(), None, None, None, None, None)
    assert ex.lib.msc_gated_ffn_backward(ex.ctx, C.byref(f), 16, 64, p, C.c_void_p(dy.data_ptr()), C.byref(part),
                                         C.c_void_p(ws.data_ptr()), ws.numel(), None) == -1
    assert ex.check() == 0


def norm64(v, nrm):
    if nrm is None:
        return v
    if nrm["kind"] == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + nrm["eps"])
    v = v * nrm["w"].double() if nrm.get("w") is not None else v
    return v + nrm["b"].double() if nrm.get("b") is not None else v


def make_stack(seed, n, c, hidden, dtype, nsamples):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape, s=1.0, m=0.0):
        return torch.randn(shape, generator=gen, device="cuda") * s + m
    blocks = []
    for i in range(3):
        _, _, ffn = make(seed + i + 1, 1, c, hidden + 8 * i, dtype, i != 1)
        blocks.append(dict(ffn=ffn, act=("silu", "gelu", "gelu_erf")[i],
                           pre=dict(kind="layer", w=r(c, s=0.1, m=1.0), b=r(c, s=0.1), eps=1e-6) if i < 2 else
                           dict(kind="rms", w=r(c, s=0.1, m=1.0), eps=1e-5),
                           post=None if i == 0 else dict(kind="rms", w=r(c, s=0.1, m=1.0), eps=1e-6),
                           gate=r(nsamples, c, s=0.3) if nsamples else r(c, s=0.3), res_scale=1.0 if i else 0.8))
    coords = torch.zeros(n, 4, dtype=torch.int32, device="cuda")
    if nsamples:
        coords[:, 3] = torch.sort(torch.randint(0, nsamples, (n,), generator=gen, device="cuda")).values
    return r(n, c), blocks, coords


@pytest.mark.parametrize("x_dtype,dtype", [(torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("n,nsamples", [(1, 0), (777, 3)])
def test_stack(ex, x_dtype, dtype, n, nsamples):
    """Three blocks in one call.  Each block rounds its normalised input, its
    hidden values and its output to 16 bits: three roundings of relative u on
    a branch whose gate is ~0.3, over 3 blocks, on a stream of order one:
    rel-L2 below 3 * 3 * u (and one rounding of a 16-bit stream a block)."""
    x, blocks, coords = make_stack(40 + n, n, 128, 344, dtype, nsamples)
    x = x.to(x_dtype)
    want = x.double()
    for b in blocks:
        h = norm64(want, b["pre"])
        w = {k: v.double() for k, v in b["ffn"].items()}
        g, u = h @ w["w_gate"].T + w.get("b_gate", 0.0), h @ w["w_up"].T + w.get("b_up", 0.0)
        f = act64(g, b["act"])[0] * u @ w["w_down"].T + w.get("b_down", 0.0)
        gate = b["gate"].double()
        want = b["res_scale"] * want + (gate[coords[:, 3].long()] if nsamples else gate) * norm64(f, b["post"])
    got = x.clone()
    ex.ffn_stack(got, blocks, coords=coords if nsamples else None)
    ex.check()
    u = torch.finfo(dtype).eps / 2
    rel = ((got.double() - want).norm() / want.norm()).item()
    assert rel <= 9 * u + (3 * u if x_dtype == dtype else 0.0), rel


def test_stack_is_the_operators_in_turn(ex):
    """One call equals norm, block, norm, ... bit for bit, and a padded batch
    leaves the rows behind it as they were."""
    x, blocks, coords = make_stack(50, 513, 64, 128, torch.bfloat16, 2)
    buf = torch.full((600, 64), 7.0, device="cuda")
    buf[:513] = x
    ex.ffn_stack(buf[:513], blocks, coords=coords)
    _, h = ex.residual_norm(x, pre=blocks[0]["pre"], branch_dtype=torch.bfloat16)
    for i, b in enumerate(blocks):
        f = ex.gated_ffn(h, b["ffn"], act=b["act"])
        nxt = blocks[i + 1]["pre"] if i < 2 else None
        x, h = ex.residual_norm(x, f, post=b["post"], gate=b["gate"], pre=nxt, res_scale=b["res_scale"], coords=coords)
    ex.check()
    assert torch.equal(buf[:513], x) and (buf[513:] == 7.0).all()


@pytest.mark.parametrize("x_dtype", [torch.float32, torch.bfloat16])
def test_stack_of_post_norm_blocks(ex, x_dtype):
    """Blocks without a pre norm (the block sees the stream in its own type)
    and without a gate.  The stream is rounded to 16 bits before each block
    (u), the hidden values and the branch once each: 3 u a block of a branch of
    order one on a stream of order one, 2 blocks, plus the 16-bit stream's."""
    x, blocks, _ = make_stack(80, 333, 72, 136, torch.bfloat16, 0)
    blocks = [{**b, "pre": None, "gate": None, "res_scale": 1.0,
               "post": dict(kind="layer", w=None, b=None, eps=1e-6)} for b in blocks[:2]]
    x = x.to(x_dtype)
    want = x.double()
    for b in blocks:
        w = {k: v.double() for k, v in b["ffn"].items()}
        h = want
        g, u = h @ w["w_gate"].T + w.get("b_gate", 0.0), h @ w["w_up"].T + w.get("b_up", 0.0)
        want = want + norm64(act64(g, b["act"])[0] * u @ w["w_down"].T + w.get("b_down", 0.0), b["post"])
    got = ex.ffn_stack(x.clone(), blocks)
    ex.check()
    rel = ((got.double() - want).norm() / want.norm()).item()
    # a relative error of the branch's input passes through the block with a
    # factor of at most two (gate and up each carry it once)
    assert rel <= 2 * 2 * 3 * 2.0 ** -8, rel


def test_stack_refused_before_it_starts(ex):
    x, blocks, coords = make_stack(60, 40, 64, 128, torch.bfloat16, 2)
    before = x.clone()
    with pytest.raises(MscError):
        ex.ffn_stack(x, blocks[:2] + [{**blocks[2], "pre": dict(kind="rms", eps=0.0)}], coords=coords)
    with pytest.raises(MscError, match="samples"):
        ex.ffn_stack(x, [blocks[0], {**blocks[1], "gate": blocks[1]["gate"][0].contiguous()}], coords=coords)
    with pytest.raises(MscError, match="coordinates"):
        ex.ffn_stack(x, blocks)
    assert torch.equal(x, before)
    assert ex.ffn_stack(x, []) is x
    assert ex.ffn_stack(x[:0].contiguous(), blocks, coords=coords[:0].contiguous()).shape == (0, 64)


@pytest.mark.parametrize("n,c,hidden", [(16900000, 128, 64), (8500000, 256, 64)])
def test_offsets_past_32_bits(ex, n, c, hidden):
    """More than 2^31 elements: the last rows, and rows around the 2^31st
    element, of the single kernel, the CTA pairs and the backward pass."""
    _, _, ffn = make(90, 1, c, hidden, torch.bfloat16, True)
    x = torch.empty(n, c, dtype=torch.bfloat16, device="cuda").normal_()
    picks = [slice(0, 200), slice(2 ** 31 // c - 100, 2 ** 31 // c + 100), slice(n - 200, n)]
    y = ex.gated_ffn(x, ffn)
    ex.check()
    for p in picks:
        want, bound = fwd_bound(x[p], ffn, "silu", torch.bfloat16)
        check(y[p], want, bound, f"y {p}")
    del y
    if c == 256:
        dy = torch.empty_like(x).normal_()
        got = ex.gated_ffn_backward(x, dy, ffn, weights=False)
        ex.check()
        for p in picks:
            want, bound = bwd_reference(x[p], dy[p], ffn, "silu", torch.bfloat16)
            check(got["x"][p], want["x"], bound["x"], f"dx {p}")
    torch.cuda.empty_cache()
