"""Feed-forward blocks at the edges of their range: gates far from zero beside
ordinary ones, stacks of mixed hidden sizes, long sums, calls in place.  The
64-bit formulas and the bound of an element are those of test_ffn_gpu."""
import math

import pytest
import torch

from test_ffn_gpu import act64, bwd_reference, check, fwd_bound, make

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -23


def at_gates(ex, g, act):
    """act(g) and act'(g) in fp32, through the public backward pass: one row
    with dh = 1 and up = 1, whose gates are the bias itself, has db_gate =
    act'(g) and db_up = act(g), both unrounded."""
    hidden = g.numel()
    zero = torch.zeros(hidden, 8, device="cuda", dtype=torch.bfloat16)
    ffn = dict(w_gate=zero, w_up=zero, w_down=torch.ones(8, hidden, device="cuda", dtype=torch.bfloat16),
               b_gate=g, b_up=torch.ones(hidden, device="cuda"))
    x = torch.zeros(1, 8, device="cuda", dtype=torch.bfloat16)
    dy = x.clone()
    dy[0, 0] = 1.0
    got = ex.gated_ffn_backward(x, dy, ffn, act=act)
    ex.check()
    return got["b_up"].double(), got["b_gate"].double()


def gate_slope64(g, act):
    """sigma's argument of the activation, its slope and exponent (64 bits)."""
    if act == "silu":
        return torch.ones_like(g), g / math.log(2)
    k = 2 * math.sqrt(2 / math.pi)
    return k * (1 + 3 * 0.044715 * g * g), k * (g + 0.044715 * g ** 3) / math.log(2)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_erf"])
@pytest.mark.parametrize("far", [6.0, 10.0, 30.0, 100.0, 1e3, 1e4, 3e5, 1e10, 1e30])
def test_large_gates_beside_ordinary_ones(ex, act, far):
    """Two neighbouring units share a reciprocal: the derivative at a large
    gate is one whatever stands beside it, and the neighbour's is its own.

    dv = s + v (1 - s) slope in fp32: s within 4 units in the last place; e =
    2^a, of which 1 - s = e s is made, within (4 + 2 |a|) units (the argument's
    two roundings and ex2's error, in units of a; counted up to a = 126, beyond
    which e is zero on both sides but for 2^-126); v and the slope within 4
    each.  The erf form's e^(-g^2 / 2) and polynomial: 1.5e-7 in erf, and the
    density's (8 + g^2) units."""
    partners = torch.linspace(-3.0, 3.0, 4096, device="cuda")
    for flip in (False, True):
        pair = [torch.full_like(partners, far), partners]
        g = torch.stack(pair[::-1] if flip else pair, 1).reshape(-1).contiguous()
        v, dv = at_gates(ex, g, act)
        g = g.double()
        if act == "gelu_erf":
            want_v, want_dv = act64(g, act)
            density = torch.exp(-g * g / 2) * g.abs()
            bound_v = 2e-7 * g.abs().clamp(max=6.0) + 8 * F32 * want_v.abs()
            bound_dv = 1e-7 + 8 * F32 + (8 + g * g) * F32 * density
        else:
            # tanh of a number this large is one, and 1 - s zero, in 64 bits too
            gc = g.clamp(max=40.0)
            slope, a = gate_slope64(gc, act)
            s = torch.sigmoid(a * math.log(2))
            rest = torch.sigmoid(-a * math.log(2))
            want_v, want_dv = g * s, s + gc * s * rest * slope
            bound_v = (8 + 2 * a.abs().clamp(max=126) * rest) * F32 * want_v.abs() + 1e-30
            bound_dv = 8 * F32 * s + (16 + 2 * a.abs().clamp(max=126)) * F32 * (gc * s * rest * slope).abs() + 1e-30
        assert v.isfinite().all() and dv.isfinite().all()
        worst = ((v - want_v).abs() / bound_v).max().item(), ((dv - want_dv).abs() / bound_dv).max().item()
        assert worst[0] <= 1.0 and worst[1] <= 1.0, (act, far, worst)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_erf"])
def test_gates_far_below_zero(ex, act):
    """Far below zero the value and the derivative are nothing, however far:
    SiLU ends at 43 2^-62 < 1e-17 (its exact value there is 9e-18), GELU below,
    the erf form at the 1.5e-7 / 2 |g| of its polynomial at most and at exactly
    zero from 20 on.  The neighbour's are its own, beside NaN and infinity too."""
    partners = torch.linspace(-3.0, 3.0, 512, device="cuda")
    alone = at_gates(ex, partners, act)
    for far in (-45.0, -60.0, -300.0, -1e4, -1e10, -1e20, -1e30, -3e38, float("-inf"), float("inf"), float("nan")):
        g = torch.stack([torch.full_like(partners, far), partners], 1).reshape(-1).contiguous()
        v, dv = at_gates(ex, g, act)
        if math.isfinite(far):
            assert v[::2].abs().max() <= 1e-17 and dv[::2].abs().max() <= 1e-15, far
        if math.isnan(far):
            assert v[::2].isnan().all() and dv[::2].isnan().all()
        # a reciprocal shared with another partner: a few units in the last
        # place (of one half in the erf form's distribution function)
        near = 8 * F32 * alone[0].abs() + (4 * F32 * partners.abs() if act == "gelu_erf" else 0.0) + 1e-30
        assert ((v[1::2] - alone[0]).abs() <= near).all(), far
        assert ((dv[1::2] - alone[1]).abs() <= 16 * F32).all(), far


def test_no_rows(ex):
    """Every call without rows: an empty dx alone, and a gate of no samples
    where there is no row to look one up."""
    x, dy, ffn = make(5, 8, 64, 128, torch.bfloat16, True)
    none = x[:0].contiguous()
    got = ex.gated_ffn_backward(none, none, ffn, weights=False)
    assert set(got) == {"x"} and got["x"].shape == (0, 64)
    gate, coords = torch.zeros(0, 64, device="cuda"), torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    r, h = ex.residual_norm(none, none, gate=gate, coords=coords, pre=dict(kind="rms", eps=1e-6))
    assert r.shape == h.shape == (0, 64)
    got = ex.residual_norm_backward(none, none, none, none, gate=gate, coords=coords, pre=dict(kind="rms", eps=1e-6))
    assert got["gate"].shape == (0, 64) and got["x"].shape == got["f"].shape == (0, 64)
    assert ex.ffn_stack(none, [dict(ffn=ffn, gate=gate)], coords=coords) is none
    assert ex.check() == 0


@pytest.mark.parametrize("n,c,sizes", [(300, 512, (1536, 1600)), (64, 256, (1600, 1536)), (8, 128, (16384, 16392))])
def test_stack_of_mixed_hidden_sizes(ex, n, c, sizes):
    """Blocks of which the smaller one needs the larger workspace, in one
    call: the operators in turn, bit for bit."""
    nrm = dict(kind="rms", eps=1e-6)
    blocks = [dict(ffn=make(i, 1, c, h, torch.bfloat16, True)[2], pre=nrm) for i, h in enumerate(sizes)]
    x = make(9, n, c, 8, torch.bfloat16, False)[0].float()
    want, h = ex.residual_norm(x, pre=nrm, branch_dtype=torch.bfloat16)
    for i, b in enumerate(blocks):
        want, h = ex.residual_norm(want, ex.gated_ffn(h, b["ffn"]), pre=nrm if i == 0 else None)
    got = ex.ffn_stack(x.clone(), blocks)
    ex.check()
    assert torch.equal(got, want)


# (rows, channels): CTA pairs of 256 columns, single CTAs, CTA pairs of 128 columns (backward: the forward
# pass of that many rows and few channels is one kernel, whose chain is the whole hidden size)
@pytest.mark.parametrize("n,c", [(9500, 1024), (4900, 512), (20000, 128)])
def test_long_sums_do_not_drift(ex, n, c):
    """65,536 hidden units, terms of one sign.  The tensor core truncates its
    fp32 accumulator: a step of 8 elements loses up to 2^-23 of the sum so far,
    which averages half of the total, so that a chain of 32,768 drifts by
    32768 / 8 * 2^-23 / 2 = 2.4e-4 at most, and one of 65,536 (y in the single
    kernel; before the limit also dx, whose dg half of the chain is small here)
    by 4.9e-4.  The mean over 64 x c outputs takes their 16-bit rounding out
    (2^-11 / sqrt(3 * 64 c) < 4e-6)."""
    hidden = 65536
    gen = torch.Generator(device="cuda").manual_seed(n)

    def positive(*shape, scale):
        return ((1.0 + torch.rand(shape, generator=gen, device="cuda")) * scale).half()
    # gates of 40: act(g) = 40, act' = 1; h = 1 for y, dg and du one sum of w_down times 1 / 40 and 1 for dx
    up = torch.full((hidden,), 1 / 40, device="cuda")
    ffn = dict(w_gate=positive(hidden, c, scale=2.0 ** -8), w_up=positive(hidden, c, scale=2.0 ** -8),
               w_down=positive(c, hidden, scale=2.0 ** -8), b_gate=torch.full((hidden,), 40.0, device="cuda"), b_up=up)
    x = torch.zeros(n, c, device="cuda", dtype=torch.float16)
    y = ex.gated_ffn(x, ffn)
    ex.check()
    h = torch.full((hidden,), 40.0 * up[0].double().item(), device="cuda", dtype=torch.float16).double()
    drift = (y[:64].double() / (ffn["w_down"].double() @ h) - 1).mean().item()
    assert abs(drift) <= (4.8e-4 if c <= 128 else 2.4e-4), drift
    dy = torch.full((n, c), 2.0 ** -6, device="cuda", dtype=torch.float16)
    dx = ex.gated_ffn_backward(x, dy, ffn, weights=False)["x"]
    ex.check()
    dh = ffn["w_down"].double().sum(0) * 2.0 ** -6
    dg, du = (dh * up[0].double()).half().double(), (dh * 40.0).half().double()
    want = dg @ ffn["w_gate"].double() + du @ ffn["w_up"].double()
    drift = (dx[:64].double() / want - 1).mean().item()
    assert abs(drift) <= 2.4e-4, drift
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,c", [(9500, 264), (4900, 512)])
def test_long_sums(ex, n, c):
    """The same parts of a long sum on random data, rows of the first and the
    last tile: every element within its bound, and the same bits again."""
    x, dy, ffn = make(n, n, c, 65536, torch.bfloat16, True)
    y = ex.gated_ffn(x, ffn)
    dx = ex.gated_ffn_backward(x, dy, ffn, weights=False)["x"]
    ex.check()
    assert torch.equal(y, ex.gated_ffn(x, ffn))
    for p in (slice(0, 40), slice(n - 40, n)):
        want, bound = fwd_bound(x[p], ffn, "silu", torch.bfloat16)
        check(y[p], want, bound, f"y {p}")
        want, bound = bwd_reference(x[p], dy[p], ffn, "silu", torch.bfloat16)
        check(dx[p], want["x"], bound["x"], f"dx {p}")
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,c,hidden", [(40000, 1024, 2048), (40000, 512, 2048), (70000, 72, 200)])
def test_weight_gradients_of_many_rows(ex, n, c, hidden):
    """More than 32,768 rows: the weight gradients' sums in two and three
    parts, on CTA pairs and on single CTAs."""
    x, dy, ffn = make(n + c, n, c, hidden, torch.bfloat16, True)
    got = ex.gated_ffn_backward(x, dy, ffn)
    ex.check()
    want, bound = bwd_reference(x, dy, ffn, "silu", torch.bfloat16)
    for k in got:
        check(got[k], want[k], bound[k], k)
    again = ex.gated_ffn_backward(x, dy, ffn)
    assert all(torch.equal(got[k], again[k]) for k in got)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,c,hidden", [(1, 1024, 2048), (7, 128, 344), (300, 264, 520), (19001, 64, 176), (19500, 128, 344),
                                        (10000, 264, 520)])
def test_in_place_on_every_path(ex, n, c, hidden):
    """y is x: the dot products, single CTAs with a K split, the single kernel
    of either width, CTA pairs."""
    x, _, ffn = make(n, n, c, hidden, torch.bfloat16, True)
    want = ex.gated_ffn(x, ffn)
    y = x.clone()
    assert ex.gated_ffn(y, ffn, out=y) is y and torch.equal(y, want)
    ex.check()
