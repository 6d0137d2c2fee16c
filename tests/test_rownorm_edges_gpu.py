"""Residual norms at the edges: rows that one column dominates, outputs in the
place of inputs, long runs of rows.  Formulas in 64 bits as in
test_rownorm_gpu."""
import ctypes as C
import math

import pytest
import torch

from mogecpp_b200 import lib as L
from test_rownorm_gpu import CHANNELS, backward64, forward64, make, norm64

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -23


def depth(c):
    """Additions that one value passes through in a row's sum: at most 16
    columns a thread (two halves of a pair each), the lanes and warps of the
    row, and a handful of roundings of the normalised value itself."""
    return 16 + math.log2(c) + 16


def dominated(seed, c):
    """c rows of order one: in row j column j is 40 sqrt(c) large."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randn(c, c, generator=gen, device="cuda")
    v.diagonal().fill_(40.0 * c ** 0.5)
    return v


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("c", CHANNELS)
def test_every_column_counts(ex, c, kind):
    """A column left out of a sum, or counted twice, changes the row's scale
    by tens of percent (the square of the large one is 1600 times the others'
    sum) or its mean by 40 / sqrt(c).

    Bounds.  The sums are off by depth 2^-24 of their absolute sums: the mean
    by depth 2^-24 mean|v|, the mean square by depth 2^-24 of itself and, with
    the centred values' own rounding 2^-24 |mean|, the scale by half of that
    each, and rsqrt by 2 units.  So |d hat| <= depth 2^-24 (|hat| + k mean|v|)
    twice over.  Backward, of k (d - mean d - hat mean(d hat)): the same depth
    on each term over absolute values, hat's own error in the last two."""
    x = dominated(c, c)
    n = x.shape[0]
    nrm = dict(kind=kind, w=None, b=None, eps=1e-6)
    zero = torch.zeros_like(x)
    e = depth(c) * F32
    hat, k = norm64(x, nrm)
    bound = e * (hat.abs() + k * x.double().abs().mean(1, keepdim=True)) + 1e-12
    _, h = ex.residual_norm(x, pre=nrm)
    r, _ = ex.residual_norm(zero, x, post=nrm)
    ex.check()
    for got in (h, r):
        assert ((got.double() - hat).abs() <= bound).all(), ((got.double() - hat).abs() / bound).max().item()
    gen = torch.Generator(device="cuda").manual_seed(c + 1)
    d = torch.randn(n, c, generator=gen, device="cuda")
    da = d.double().abs()
    mean = da.mean(1, keepdim=True) if kind == "layer" else 0.0
    size = k * (da + mean + hat.abs() * (da * hat.abs()).mean(1, keepdim=True))
    # hat's error times |d|, summed, meets hat once more; and hat's own in the outer product
    extra = k * ((da * bound).mean(1, keepdim=True) * hat.abs() + bound * (da * hat.abs()).mean(1, keepdim=True))
    tol = 2 * e * size + 2 * extra + 1e-12
    zeros = torch.zeros_like(x)
    want = backward64(x, None, None, d, dict(pre=nrm, post=None, gate=None, coords=None), 1.0)[0]["x"]
    got = ex.residual_norm_backward(x, None, None, d, pre=nrm)["x"]
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol).max().item()
    got = ex.residual_norm_backward(zeros, x, d, None, post=nrm)["f"]
    ex.check()
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs() / tol).max().item()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,c", [(1, 8), (1237, 64), (5000, 128), (900, 512), (300, 2056)])
@pytest.mark.parametrize("x_dtype,f_dtype", [(torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16)])
def test_outputs_in_the_place_of_inputs(ex, n, c, x_dtype, f_dtype):
    """r is x and h is f; dx is dr and df is dh, through the C call: the same
    bits as with outputs of their own."""
    x, f, dr, dh, cfg = make(n + c, n, c, x_dtype, f_dtype, "rms", "layer", "sample", order="shuffled")
    want_r, want_h = ex.residual_norm(x, f, res_scale=0.7, **cfg)
    d = ex._residual(n, c, x_dtype, f_dtype, cfg["post"], cfg["gate"], cfg["pre"], 0.7, cfg["coords"])
    r, h = x.clone(), f.clone()
    L.check(ex.lib.msc_residual_norm(ex.ctx, C.byref(d), n, r.data_ptr(), h.data_ptr(), cfg["coords"].data_ptr(),
                                     r.data_ptr(), h.data_ptr(), ex._raw_stream()))
    ex.check()
    assert torch.equal(r, want_r) and torch.equal(h, want_h)
    want = ex.residual_norm_backward(want_r, f, dr, dh, res_scale=0.7, **cfg)
    a, b = dr.clone(), dh.clone()
    g = L.ResidualNormGrads(a.data_ptr(), b.data_ptr(), None, None, None, None, None)
    ws = ex._scratch(x, ex.lib.msc_residual_norm_backward_workspace_bytes(n, c, d.nsamples))
    L.check(ex.lib.msc_residual_norm_backward(ex.ctx, C.byref(d), n, r.data_ptr(), f.data_ptr(), cfg["coords"].data_ptr(),
                                              a.data_ptr(), b.data_ptr(), C.byref(g), ws.data_ptr(), ws.numel(),
                                              ex._raw_stream()))
    ex.check()
    assert torch.equal(a, want["x"]) and torch.equal(b, want["f"])


@pytest.mark.parametrize("spread", ["sorted", "shuffled", "one"])
@pytest.mark.parametrize("n,c,nsamples", [(300000, 128, 32768), (200000, 64, 32768), (30000, 1024, 16000)])
def test_long_runs_of_rows(ex, n, c, nsamples, spread):
    """Many samples leave few units with long runs of rows.  Terms of one sign
    whose every addition would round the same way (1/3 next to a large sum):
    one fp32 chain over a unit's rows is off by up to 1e-3, runs of 1,024 steps
    by (1024 + 16) 2^-24 of the sum at most (a term's own error, from the norm
    of a constant gradient, adds 64 2^-24); a sample's gate is added up likewise,
    one fp32 addition per change of sample besides."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    r = torch.randn(n, c, generator=gen, device="cuda")
    third = torch.full((n, c), 1 / 3, device="cuda")
    s = torch.randint(0, nsamples, (n,), generator=gen, device="cuda")
    s = torch.sort(s).values if spread == "sorted" else (s if spread == "shuffled" else s * 0 + 5)
    coords = torch.zeros(n, 4, dtype=torch.int32, device="cuda")
    coords[:, 3] = s
    one, zero = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    nrm = dict(kind="layer", w=one, b=one, eps=1e-6)
    gate = torch.ones(nsamples, c, device="cuda")
    got = ex.residual_norm_backward(r, torch.zeros_like(r), third, third, post=nrm, gate=gate, coords=coords,
                                    pre=dict(nrm, b=zero))
    ex.check()
    t = third[0, 0].double().item()
    rows = torch.bincount(s, minlength=nsamples).double()
    u = 2.0 ** -24
    limit = (1024 + 16 + 64) * u
    for k in ("pre_b", "post_b"):
        assert ((got[k].double() - n * t).abs() <= limit * n * t).all(), (k, ((got[k].double() / (n * t)) - 1).abs().max().item())
    # f^ is zero, so that t is the post norm's bias, one
    off = (got["gate"].double() - rows[:, None] * t).abs()
    assert (off <= (limit + u * rows[:, None].clamp(max=1024)) * rows[:, None] * t + 1e-30).all()
    hat, _ = norm64(r, nrm)
    want, size = (t * hat).sum(0), (t * hat).abs().sum(0)
    assert ((got["pre_w"].double() - want).abs() <= (limit + depth(c) * F32) * size).all()
    torch.cuda.empty_cache()
