"""Residual norms (norm after a block, gate, residual scale, norm before the
next), forward and backward, against plain 64-bit formulas.

Tolerances.  Everything between the loads and the one rounding of each output
is fp32: a mean over c values is off by at most c 2^-24 of the mean absolute
value (pairwise in practice), the scale by a few ulp, so a normalised value is
within (c + 32) 2^-24 times (|v^| + the row's largest |v|/std); for rows of
order one that is bounded by (c + 32) 2^-23 (1 + |v^|) with room.  A 16-bit
output adds u = eps / 2 of itself.  Column sums add n values of relative error
as above in fp32 runs, then double."""
import pytest
import torch

from mogecpp_b200.lib import MscError

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -23


def make(seed, n, c, x_dtype, f_dtype, post, pre, gate, nsamples=3, order="sorted"):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape, s=1.0, m=0.0):
        return torch.randn(shape, generator=gen, device="cuda") * s + m

    def nrm(kind):
        if kind is None:
            return None
        return dict(kind=kind, w=r(c, s=0.1, m=1.0), b=r(c, s=0.1) if kind == "layer" else None, eps=1e-6)
    coords = torch.zeros(n, 4, dtype=torch.int32, device="cuda")
    s = torch.randint(0, nsamples, (n,), generator=gen, device="cuda")
    coords[:, 3] = torch.sort(s).values if order == "sorted" else s
    g = {"none": None, "channel": r(c, s=0.3, m=0.5), "sample": r(nsamples, c, s=0.3, m=0.5)}[gate]
    cfg = dict(post=nrm(post), pre=nrm(pre), gate=g, coords=coords if gate == "sample" else None)
    return (r(n, c, s=1.3, m=0.2).to(x_dtype), r(n, c, s=0.8, m=-0.1).to(f_dtype), r(n, c, s=0.3).to(x_dtype),
            r(n, c, s=0.3).to(f_dtype), cfg)


def norm64(v, nrm):
    v = v.double()
    if nrm["kind"] == "layer":
        v = v - v.mean(1, keepdim=True)
    k = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + nrm["eps"])
    return v * k, k


def aff(v, nrm):
    v = v * nrm["w"].double() if nrm["w"] is not None else v
    return v + nrm["b"].double() if nrm["b"] is not None else v


def gate_rows(cfg):
    g = cfg["gate"]
    if g is None:
        return 1.0
    return g.double() if cfg["coords"] is None else g.double()[cfg["coords"][:, 3].long()]


def forward64(x, f, cfg, s):
    t = f.double() if cfg["post"] is None else aff(norm64(f, cfg["post"])[0], cfg["post"])
    r = s * x.double() + gate_rows(cfg) * t
    return r, None if cfg["pre"] is None else aff(norm64(r, cfg["pre"])[0], cfg["pre"])


def close(got, want, c, what, extra=0.0):
    u = torch.finfo(got.dtype).eps / 2
    tol = u * want.abs() + (c + 32) * F32 * (1 + want.abs()) + 2.0 ** -25 + extra
    worst = ((got.double() - want).abs() / tol).max().item() if want.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst} of the bound"


TYPES = [(torch.float32, torch.float32), (torch.float32, torch.float16), (torch.float32, torch.bfloat16),
         (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)]
# every row layout (8 to 512 threads a row), channels that leave threads without a column
CHANNELS = [8, 56, 64, 72, 128, 136, 256, 264, 512, 520, 1000, 1024, 2048, 2056, 4104, 8192]


@pytest.mark.parametrize("c", CHANNELS)
@pytest.mark.parametrize("x_dtype,f_dtype", TYPES)
def test_forward(ex, c, x_dtype, f_dtype):
    for n, post, pre, gate, s in ((1, "rms", "layer", "channel", 1.0), (37, "layer", "rms", "sample", 0.7),
                                  (130, None, "layer", "none", 1.0), (5, "layer", None, "sample", 0.5)):
        x, f, _, _, cfg = make(c + n, n, c, x_dtype, f_dtype, post, pre, gate)
        r, h = ex.residual_norm(x, f, res_scale=s, **cfg)
        ex.check()
        want_r, want_h = forward64(x, f, cfg, s)
        close(r, want_r, c, f"r {n}")
        if pre is None:
            assert h is None
        else:
            close(h, want_h, c, f"h {n}")


def backward64(r, f, dr, dh, cfg, s):
    """The written-out gradients (no autograd)."""
    def back(d, hat, k, nrm):
        d = d * nrm["w"].double() if nrm["w"] is not None else d
        if nrm["kind"] == "layer":
            d = d - d.mean(1, keepdim=True)
        return k * (d - hat * (d * hat).mean(1, keepdim=True))
    out, mag = {}, {}

    def cols(k, v):
        out[k], mag[k] = v.sum(0), v.abs().sum(0)
    g = dr.double() if dr is not None else torch.zeros_like(r, dtype=torch.float64)
    if cfg["pre"] is not None:
        hat, k = norm64(r, cfg["pre"])
        cols("pre_w", dh.double() * hat)
        if cfg["pre"]["b"] is not None:
            cols("pre_b", dh.double())
        g = g + back(dh.double(), hat, k, cfg["pre"])
    elif dh is not None:
        g = g + dh.double()
    out["x"] = s * g
    if f is None:
        return out, mag
    gate = gate_rows(cfg)
    t = f.double()
    if cfg["post"] is not None:
        hat, k = norm64(f, cfg["post"])
        t = aff(hat, cfg["post"])
    if cfg["gate"] is not None:
        if cfg["coords"] is None:
            cols("gate", g * t)
        else:
            out["gate"] = torch.zeros_like(cfg["gate"], dtype=torch.float64)
            out["gate"].index_add_(0, cfg["coords"][:, 3].long(), g * t)
            mag["gate"] = torch.zeros_like(out["gate"]).index_add_(0, cfg["coords"][:, 3].long(), (g * t).abs())
    dt = gate * g
    out["f"] = dt if cfg["post"] is None else back(dt, hat, k, cfg["post"])
    if cfg["post"] is not None:
        cols("post_w", dt * hat)
        if cfg["post"]["b"] is not None:
            cols("post_b", dt)
    return out, mag


def check_backward(got, want, mag, c, what):
    assert set(got) == set(want), what
    for k in got:
        if k in ("x", "f"):
            close(got[k], want[k], c, f"{what} {k}", extra=(c + 32) * F32)
        else:
            # each of the summed values carries the rows' error; fp32 runs, then double
            tol = (c + 400) * F32 * (mag[k] + 1e-3) + 1e-7
            worst = ((got[k].double() - want[k]).abs() / tol).max().item()
            assert worst <= 1.0, f"{what} {k}: {worst} of the bound"


@pytest.mark.parametrize("c", CHANNELS)
@pytest.mark.parametrize("x_dtype,f_dtype", TYPES)
def test_backward(ex, c, x_dtype, f_dtype):
    for n, post, pre, gate, s in ((1, "rms", "layer", "channel", 1.0), (37, "layer", "rms", "sample", 0.7),
                                  (130, None, "layer", "none", 1.0), (5, "layer", None, "sample", 0.5)):
        r, f, dr, dh, cfg = make(2 * c + n, n, c, x_dtype, f_dtype, post, pre, gate)
        dh = dh if pre else None
        got = ex.residual_norm_backward(r, f, dr, dh, res_scale=s, **cfg)
        ex.check()
        want, mag = backward64(r, f, dr, dh, cfg, s)
        check_backward(got, want, mag, c, f"n={n}")


@pytest.mark.parametrize("order", ["sorted", "shuffled"])
@pytest.mark.parametrize("n,c,nsamples", [(9000, 64, 2), (9001, 128, 127), (3000, 256, 5), (1500, 512, 3), (70, 40, 300)])
def test_gate_per_sample(ex, order, n, c, nsamples):
    """Samples in any order, more samples than rows, samples without a row."""
    r, f, dr, dh, cfg = make(n, n, c, torch.float32, torch.float16, "layer", "rms", "sample", nsamples, order)
    got = ex.residual_norm_backward(r, f, dr, dh, **cfg)
    ex.check()
    want, mag = backward64(r, f, dr, dh, cfg, 1.0)
    check_backward(got, want, mag, c, order)
    again = ex.residual_norm_backward(r, f, dr, dh, **cfg)
    assert all(torch.equal(got[k], again[k]) for k in got)


def test_gradient_against_differences(ex):
    """Central differences of the 64-bit forward along one direction of each
    input (x as r: the residual sum is linear in it)."""
    n, c, s = 40, 72, 0.7
    x, f, dr, dh, cfg = make(3, n, c, torch.float32, torch.float32, "layer", "rms", "sample")
    r = forward64(x, f, cfg, s)[0].float()
    # x such that r is the forward's output to fp32: the gradients are taken at that r
    got = ex.residual_norm_backward(r, f, dr, dh, res_scale=s, **cfg)
    x64 = (r.double() - forward64(torch.zeros_like(x), f, cfg, s)[0]) / s

    def loss(xx, ff, cc):
        rr, hh = forward64(xx, ff, cc, s)
        return (rr * dr.double()).sum().item() + (hh * dh.double()).sum().item()
    gen = torch.Generator(device="cuda").manual_seed(4)
    f64 = f.double()
    for k in got:
        shape = got[k].shape
        d = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64)
        d /= d.norm()

        def at(e):
            if k == "x":
                return loss(x64 + e * d, f64, cfg)
            if k == "f":
                return loss(x64, f64 + e * d, cfg)
            cc = {**cfg, "post": dict(cfg["post"]), "pre": dict(cfg["pre"])}
            if k == "gate":
                cc["gate"] = cfg["gate"].double() + e * d
            else:
                which, part = k.split("_")
                cc[which][part] = cfg[which][part].double() + e * d
            return loss(x64, f64, cc)
        diff = (at(1e-4) - at(-1e-4)) / 2e-4
        along = (got[k].double() * d).sum().item()
        # fp32 gradients of order one: (c + 400) 2^-23 of the norm, and the difference's own ~1e-7
        assert abs(along - diff) <= (c + 400) * F32 * (got[k].double().norm().item() + 1.0) + 1e-6, k


def test_entry_norm_identity_and_absent_parts(ex):
    x, f, dr, dh, cfg = make(5, 65, 128, torch.float32, torch.bfloat16, "rms", "layer", "channel")
    r, h = ex.residual_norm(x, pre=cfg["pre"], branch_dtype=torch.bfloat16)
    assert torch.equal(r, x) and h.dtype == torch.bfloat16
    close(h, aff(norm64(x, cfg["pre"])[0], cfg["pre"]), 128, "entry")
    got = ex.residual_norm_backward(x, None, None, dh, pre=cfg["pre"])
    want, mag = backward64(x, None, None, dh, dict(cfg, gate=None), 1.0)
    check_backward(got, want, mag, 128, "entry")
    # weights may be absent; in place
    plain = dict(kind="rms", w=None, b=None, eps=1e-6)
    y = x.clone()
    r, h = ex.residual_norm(y, f, post=plain, pre=plain, res_scale=0.5, in_place=True)
    assert r.data_ptr() == y.data_ptr()
    wr, wh = forward64(x, f, dict(post=plain, pre=plain, gate=None, coords=None), 0.5)
    close(r, wr, 128, "r")
    close(h, wh, 128, "h")
    g = ex.residual_norm_backward(x, f, dr, None, post=None, gate=cfg["gate"])
    want, mag = backward64(x, f, dr, None, dict(post=None, pre=None, gate=cfg["gate"], coords=None), 1.0)
    check_backward(g, want, mag, 128, "no norms")


def test_constant_zero_and_non_finite_rows(ex):
    """A row of equal values has variance zero (the scale is 1 / sqrt(eps), the
    normalised row 0); a row with infinities or NaN spoils itself alone."""
    x, f, _, _, cfg = make(6, 40, 128, torch.bfloat16, torch.bfloat16, "layer", "layer", "channel")
    f[3] = 2.0
    x[7], f[7] = 0.0, 0.0
    want = ex.residual_norm(x, f, **cfg)
    wr, wh = forward64(x, f, cfg, 1.0)
    close(want[0], wr, 128, "r")
    bad = f.clone()
    bad[11] = float("inf")
    bad[12, 3] = float("nan")
    got = ex.residual_norm(x, bad, **cfg)
    keep = [i for i in range(40) if i not in (11, 12)]
    for a, b in zip(got, want):
        assert torch.equal(a[keep], b[keep])
        assert not a[11:13].isfinite().any()


def test_empty_and_rows_behind(ex):
    x, f, dr, dh, cfg = make(7, 100, 64, torch.bfloat16, torch.bfloat16, "rms", "rms", "sample")
    e = x[:0].contiguous()
    cfg0 = dict(cfg, coords=cfg["coords"][:0].contiguous())
    r, h = ex.residual_norm(e, e, **cfg0)
    assert r.shape == h.shape == (0, 64)
    g = ex.residual_norm_backward(e, e, e, e, **cfg0)
    assert all(not v.any() for v in g.values())
    buf = torch.full((120, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    buf[:100] = x
    r, _ = ex.residual_norm(buf[:100], f, in_place=True, **cfg)
    assert torch.equal(r, ex.residual_norm(x, f, **cfg)[0]) and (buf[100:] == 5.0).all()


def test_bad_sample_index(ex):
    """A sample outside the gate's rows is a device failure reported by check;
    the row keeps its residual alone."""
    x, f, dr, dh, cfg = make(8, 50, 64, torch.float32, torch.float16, "rms", "rms", "sample")
    good, _ = ex.residual_norm(x, f, **cfg)
    for bad in (-1, 3, 1 << 30):
        c2 = dict(cfg, coords=cfg["coords"].clone())
        c2["coords"][20, 3] = bad
        r, _ = ex.residual_norm(x, f, **c2)
        with pytest.raises(MscError, match="coordinate-out-of-range"):
            ex.check()
        assert torch.equal(r[20], x[20])
        keep = [i for i in range(50) if i != 20]
        assert torch.equal(r[keep], good[keep])
        got = ex.residual_norm_backward(x, f, dr, dh, **c2)
        with pytest.raises(MscError, match="coordinate-out-of-range"):
            ex.check()
        k = [i for i in range(50) if i != 20]
        c3 = dict(cfg, coords=cfg["coords"][k].contiguous())
        ref = ex.residual_norm_backward(x[k].contiguous(), f[k].contiguous(), dr[k].contiguous(), dh[k].contiguous(), **c3)
        assert (got["gate"] - ref["gate"]).abs().max().item() <= 100 * F32 * 50
        assert not got["f"][20].any()


def test_streams_and_graphs(ex):
    sets = [make(30 + i, 3000, 128, torch.bfloat16, torch.bfloat16, "layer", "rms", "sample") for i in range(2)]

    def both(r, f, dr, dh, cfg):
        a, b = ex.residual_norm(r, f, **cfg)
        return [a, b] + list(ex.residual_norm_backward(r, f, dr, dh, **cfg).values())
    want = [both(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(both(*s))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))
    graphs, outs = [], []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(both(*s))
        graphs.append(gr)
    for _ in range(3):
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))


def test_refusals(ex):
    x, f, dr, dh, cfg = make(9, 20, 64, torch.float16, torch.float16, "rms", "layer", "sample")
    with pytest.raises(MscError, match="residual stream"):
        ex.residual_norm(x, f.float(), **cfg)
    with pytest.raises(MscError, match="coordinates"):
        ex.residual_norm(x, f, **dict(cfg, coords=None))
    with pytest.raises(MscError, match="kind"):
        ex.residual_norm(x, f, pre=dict(kind="batch", eps=1e-6))
    with pytest.raises(MscError, match="eps"):
        ex.residual_norm(x, f, pre=dict(kind="rms", eps=0.0))
    with pytest.raises(MscError, match="norm w"):
        ex.residual_norm(x, f, pre=dict(kind="rms", w=torch.ones(32, device="cuda"), eps=1e-6))
    with pytest.raises(MscError, match="gate"):
        ex.residual_norm(x, f, gate=torch.ones(64, device="cuda", dtype=torch.float16))
    with pytest.raises(MscError, match="coords"):
        ex.residual_norm(x, f, **dict(cfg, coords=cfg["coords"].long()))
    with pytest.raises(MscError, match="multiple of 8"):
        ex.residual_norm(x[:, :60].contiguous(), f[:, :60].contiguous())
    with pytest.raises(MscError, match="f must be"):
        ex.residual_norm(x, f[:10].contiguous())
    with pytest.raises(MscError, match="contiguous"):
        ex.residual_norm(x.t().contiguous().t(), f)
    with pytest.raises(MscError, match="dh"):
        ex.residual_norm_backward(x, f, dr, None, **cfg)
    with pytest.raises(MscError, match="no gradient"):
        ex.residual_norm_backward(x, f, None, None)
    assert ex.check() == 0


def test_offsets_past_32_bits(ex):
    """More than 2^31 elements: rows at the start, around the 2^31st element
    and at the end, and a column sum over all of them."""
    n, c = 34000000, 64
    _, _, _, _, cfg = make(40, 1, c, torch.bfloat16, torch.bfloat16, "rms", "layer", "channel")
    x = torch.empty(n, c, dtype=torch.bfloat16, device="cuda").normal_()
    f = torch.empty_like(x).normal_()
    picks = [slice(0, 100), slice(2 ** 31 // c - 50, 2 ** 31 // c + 50), slice(n - 100, n)]
    r, h = ex.residual_norm(x, f, **cfg)
    ex.check()
    for p in picks:
        wr, wh = forward64(x[p], f[p], cfg, 1.0)
        close(r[p], wr, c, f"r {p}")
        close(h[p], wh, c, f"h {p}")
    got = ex.residual_norm_backward(x, f, r, h, **cfg)
    ex.check()
    for p in picks:
        want, _ = backward64(x[p], f[p], r[p], h[p], cfg, 1.0)
        for k in ("x", "f"):
            close(got[k][p], want[k], c, f"{k} {p}", extra=(c + 32) * F32)
    total = sum(h[i:i + 1000000].double().sum(0) for i in range(0, n, 1000000))
    size = sum(h[i:i + 1000000].double().abs().sum(0) for i in range(0, n, 1000000))
    # a warp adds ~14,000 rows in fp32 (each addition 2^-24 of the sum so far,
    # which grows like the root of the rows), then double
    assert ((got["pre_b"].double() - total).abs() <= 14500 * 2.0 ** -24 * size).all()
    torch.cuda.empty_cache()
