"""The language-model operators on the device against their definitions in 64 bits.

Tolerances.  u = 2^-24 is the unit of an fp32 operation; a store rounds by at most half a
step, half(T) = eps(T) / 2 of the value (plus half a subnormal step, tiny(T), where the
result may be that small).  A sum of K products of 16-bit values has exact products and at
most K additions in any order: its error is at most 2 K u sum |a b| (the factor 2 allows
additions that truncate).  Exponentials, divisions and square roots count a few u."""
import ctypes as C

import numpy as np
import pytest

from hc_amd import runtime as rt

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half(ty):
    return torch.finfo(ty).eps / 2


def tiny(ty):
    """Half the distance of the type's smallest numbers."""
    return torch.finfo(ty).tiny * torch.finfo(ty).eps / 2


def dev(x, ty=None):
    return x.to(device="cuda", dtype=ty or x.dtype)


def empty(*shape, ty):
    """An output full of a value that no operator produces here."""
    return torch.full(shape, 77.0, device="cuda").to(ty)


def f64(x):
    return x.detach().cpu().double()


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def strided(x, pad, offset=0):
    """The same values with rows further apart, `offset` elements behind an aligned address."""
    if pad == 0 and offset == 0:
        return x
    wide = torch.full((x.shape[0], x.shape[1] + pad + offset), 55.0, device=x.device).to(x.dtype)
    wide[:, offset:offset + x.shape[1]] = x
    return wide[:, offset:offset + x.shape[1]]


def near(got, want, tol, what=""):
    got = f64(got)
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4],
                           (tol if torch.is_tensor(tol) else torch.full_like(want, tol))[bad][:4])


# ---------------------------------------------------------------------------
# add + RMS norm
# ---------------------------------------------------------------------------
NORM_SHAPES = [(1, 1), (3, 7), (5, 64), (2, 520), (70, 1000), (4, 4096), (3, 5001), (2, 8192), (5, 9000), (1, 16384), (2, 33000)]


def norm_reference(x, r, w, eps, ty):
    h = x.float() if r is None else x.float() + r.float()
    h = h.to(ty)                                        # what the operator defines as h, exactly
    hd = f64(h)
    rstd = 1 / (hd.square().mean(1, keepdim=True) + eps).sqrt()
    wd = torch.ones(1, dtype=torch.float64) if w is None else f64(w)
    return h, hd, rstd, wd


def norm_roundings(cols):
    """A sum of squares in fp32: at most cols / 64 terms in a row in one lane, and the joining of lanes; its
    relative error counts half in rstd; a division, a square root and two products follow."""
    return (cols / 64 + 20) * U


@pytest.mark.parametrize("layout", ["dense", "strided", "odd", "bare"])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("ty", TYPES)
def test_add_rms_norm(ty, shape, layout):
    rows, cols = shape
    t = TYPES[ty]
    x, r = dev(normal(1, rows, cols), t), dev(3 * normal(2, rows, cols), t)
    w = dev(1 + 0.2 * normal(3, cols), t if layout == "odd" else torch.float32)
    pad, off = {"strided": (16, 0), "odd": (3, 1)}.get(layout, (0, 0))
    if layout == "bare":
        r = w = None
    out, summed = (strided(empty(rows, cols, ty=t), pad, off) for _ in range(2))
    rstd = empty(rows, ty=torch.float32)
    rt.add_rms_norm(strided(x, pad, off), None if r is None else strided(r, pad, off), w, out, eps=1e-5,
                    summed=summed, rstd=rstd)
    h, hd, want_rstd, wd = norm_reference(x, r, w, 1e-5, t)
    assert torch.equal(summed, h)
    near(rstd, want_rstd[:, 0], norm_roundings(cols) * want_rstd[:, 0], "rstd")
    want = hd * want_rstd * wd
    near(out, want, want.abs() * (half(t) + norm_roundings(cols)) + tiny(t), "out")
    if layout in ("strided", "odd"):            # what lies between the rows stays
        assert bool((out._base[:, off + cols:] == 55).all()) and bool((out._base[:, :off] == 55).all())
        assert bool((summed._base[:, off + cols:] == 55).all())


@pytest.mark.parametrize("layout", ["dense", "strided", "odd", "bare"])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("ty", TYPES)
def test_add_rms_norm_int8(ty, shape, layout):
    rows, cols = shape
    t = TYPES[ty]
    x, r = dev(normal(1, rows, cols), t), dev(3 * normal(2, rows, cols), t)
    # powers of two and exact halves of the largest value: quotients that are ties
    x[0] = dev(torch.pow(2.0, torch.arange(cols) % 9).neg(), t)
    r[0] = 0
    w = dev(1 + 0.2 * normal(3, cols), t if layout == "odd" else torch.float32)
    pad, off = {"strided": (16, 0), "odd": (3, 1)}.get(layout, (0, 0))
    if layout == "bare":
        r = w = None
    q = torch.full((rows, cols + pad + off), 101, device="cuda", dtype=torch.int8)[:, off:off + cols]
    scale, summed = empty(rows, ty=torch.float32), empty(rows, cols, ty=t)
    rt.add_rms_norm(strided(x, pad, off), None if r is None else strided(r, pad, off), w, q, summed=summed, scale=scale)
    h, hd, rstd, wd = norm_reference(x, r, w, 1e-6, t)
    v = hd * wd
    most = v.abs().amax(1, keepdim=True)
    assert torch.equal(summed, h)
    assert torch.equal(q.cpu(), torch.where(most > 0, 127 * v / most, 0.0).round().to(torch.int8))
    want = (rstd * most / 127)[:, 0]
    near(scale, want, norm_roundings(cols) * want, "scale")
    if pad:
        assert bool((q._base[:, off + cols:] == 101).all())


@pytest.mark.parametrize("cols", [8, 100, 4096, 20000])
@pytest.mark.parametrize("ty", TYPES)
def test_add_rms_norm_special_rows(ty, cols):
    """Rows of zeros, tiny and huge values, one NaN, one infinity: each row by itself."""
    t = TYPES[ty]
    x = normal(4, 7, cols)
    x[0], x[1], x[2] = 0, 0, x[2] * 1e-30
    x[1, cols // 2] = 3.0
    x[3] *= 60000.0 / x[3].abs().max()
    x[4, 1], x[5, cols - 1] = float("nan"), float("-inf")
    x = dev(x, t)
    q, y = torch.empty(7, cols, device="cuda", dtype=torch.int8), torch.empty_like(x)
    scale = empty(7, ty=torch.float32)
    rt.add_rms_norm(x, None, None, q, eps=0.0, scale=scale)
    rt.add_rms_norm(x, None, None, y, eps=1e-6)
    xd = f64(x)
    for row in (1, 3, 6) + ((2,) if bool((xd[2] != 0).any()) else ()):
        most = xd[row].abs().max()
        assert torch.equal(q[row].cpu(), (127 * xd[row] / most).round().to(torch.int8)), row
    assert not bool(q[0].any()) and not bool(q[4].any()) and not bool(q[5].any())
    assert bool(torch.isnan(scale[4])) and bool(torch.isnan(scale[5]))
    assert not bool(y[0].any()) and bool(torch.isnan(y[4]).all())
    assert bool(torch.isfinite(y[6]).all())
    zero = empty(1, ty=torch.float32)
    rt.add_rms_norm(x[:1], None, None, q[:1], eps=1e-6, scale=zero)
    assert float(zero[0]) == 0.0


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("cols", [1000, 4096, 30001])
def test_add_rms_norm_in_place(ty, cols):
    """summed may be the residual and out may be x."""
    t = TYPES[ty]
    x, r = dev(normal(5, 9, cols), t), dev(normal(6, 9, cols), t)
    w = dev(1 + 0.2 * normal(7, cols))
    h, y = torch.empty_like(x), torch.empty_like(x)
    rt.add_rms_norm(x, r, w, y, summed=h)
    rt.add_rms_norm(x, r, w, x, summed=r)
    assert torch.equal(x, y) and torch.equal(r, h)


def norm_back_reference(dy, hd, rstd, wd, ds):
    a, n = dy * wd, hd * rstd
    return ds + rstd * (a - n * (a * n).mean(1, keepdim=True)), (dy * n).sum(0)


@pytest.mark.parametrize("layout", ["dense", "strided", "odd", "bare"])
@pytest.mark.parametrize("shape", NORM_SHAPES + [(1000, 96), (517, 2048)], ids=str)
@pytest.mark.parametrize("ty", TYPES)
def test_add_rms_norm_backward(ty, shape, layout):
    rows, cols = shape
    t = TYPES[ty]
    wt = t if layout == "odd" else torch.float32
    h, dy, ds = (dev(normal(k, rows, cols), t) for k in (1, 2, 3))
    w = dev(1 + 0.2 * normal(4, cols), wt)
    _, hd, rstd, wd = norm_reference(h, None, w, 1e-6, t)
    rstd_in = rstd[:, 0].float().cuda()
    pad, off = {"strided": (16, 0), "odd": (3, 1)}.get(layout, (0, 0))
    gx, gw = strided(empty(rows, cols, ty=t), pad, off), empty(cols, ty=wt)
    if layout == "bare":
        rt.add_rms_norm_backward(dy, h, None, rstd_in, gx)
        wd, dsd = torch.ones(1, dtype=torch.float64), torch.zeros(1, dtype=torch.float64)
    else:
        rt.add_rms_norm_backward(strided(dy, pad, off), strided(h, pad, off), w, rstd_in, gx, gw,
                                 grad_summed=strided(ds, pad, off))
        dsd = f64(ds)
    dyd = f64(dy)
    want_x, want_w = norm_back_reference(dyd, hd, rstd, wd, dsd)
    # every term carries at most the roundings of a sum of cols / 64 terms and its joining, relative to the
    # sums of magnitudes
    a, n = (dyd * wd).abs(), (hd * rstd).abs()
    size = dsd.abs() + rstd * (a + n * (a * n).mean(1, keepdim=True))
    near(gx, want_x, want_x.abs() * half(t) + size * (cols / 64 + 24) * U + tiny(t), "grad_in")
    if layout != "bare":
        near(gw, want_w, want_w.abs() * half(wt) * (wt != torch.float32) +
             (dyd.abs() * n).sum(0) * (rows + 300) * U + tiny(wt), "grad_weight")


def test_add_rms_norm_gradients_are_the_slopes():
    """Against differences of the definition in 64 bits, along random directions."""
    rows, cols = 13, 200
    x, r, w = normal(1, rows, cols), normal(2, rows, cols), 1 + 0.2 * normal(3, cols)
    dy, ds = normal(4, rows, cols), normal(5, rows, cols)

    def total(x, r, w):
        h = x + r
        return ((h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * w) * dy.double() + h * ds.double()).sum()
    xg, rg, wg = dev(x), dev(r), dev(w)
    y, h, rstd = torch.empty_like(xg), torch.empty_like(xg), empty(rows, ty=torch.float32)
    gx, gw = torch.empty_like(xg), torch.empty_like(wg)
    rt.add_rms_norm(xg, rg, wg, y, summed=h, rstd=rstd)
    rt.add_rms_norm_backward(dev(dy), h, wg, rstd, gx, gw, grad_summed=dev(ds))
    e = 1e-5
    for seed in range(3):
        dx, dw = normal(10 + seed, rows, cols).double(), normal(20 + seed, cols).double()
        for which, got in (("x", (f64(gx) * dx).sum()), ("r", (f64(gx) * dx).sum()), ("w", (f64(gw) * dw).sum())):
            step = {"x": (dx, 0, 0), "r": (0, dx, 0), "w": (0, 0, dw)}[which]
            up = total(x + e * step[0], r.double() + e * step[1], w.double() + e * step[2])
            down = total(x - e * step[0], r.double() - e * step[1], w.double() - e * step[2])
            # h is rounded to fp32 before it is normalised: at most u per element, like the other roundings
            size = (f64(gx).abs() * dx.abs()).sum() + (f64(gw).abs() * dw.abs()).sum()
            assert abs((up - down) / (2 * e) - got) <= size * 200 * U + 1e-5, which


# ---------------------------------------------------------------------------
# gated feed-forward block
# ---------------------------------------------------------------------------
FFN_SHAPES = [(1, 8, 8), (1, 1, 1), (1, 4096, 96), (2, 136, 40), (5, 1000, 77), (16, 512, 130), (17, 72, 64), (33, 333, 97),
              (64, 2048, 64), (100, 65, 129), (130, 129, 200), (257, 264, 392), (300, 1024, 257), (513, 640, 520)]


def act_reference(kind, g):
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    a, b = (2 / torch.pi) ** 0.5, 0.044715
    t = torch.tanh(a * (g + b * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * b * g * g)


def ffn_inputs(t, d, f, ty, pad=0, off=0):
    x = dev(normal(1, t, d), ty)
    wg, wu = (dev(normal(k, f, d) * d ** -0.5, ty) for k in (2, 3))
    return x, wg, wu


@pytest.mark.parametrize("layout", ["dense", "strided", "odd"])
@pytest.mark.parametrize("shape", FFN_SHAPES, ids=str)
@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_gated_ffn(ty, shape, layout):
    t, d, f = shape
    k = TYPES[ty]
    kind = "gelu" if layout == "strided" else "silu"
    x, wg, wu = ffn_inputs(t, d, f, k)
    pad, off = {"strided": (16, 0), "odd": (3, 1)}.get(layout, (0, 0))
    out, gate, up = (strided(empty(t, f, ty=k), pad, off) for _ in range(3))
    rt.gated_ffn(strided(x, pad, off), strided(wg, pad, off), strided(wu, pad, off), out, activation=kind, gate=gate, up=up)
    xd, gd, ud = f64(x), f64(wg), f64(wu)
    g, u = xd @ gd.t(), xd @ ud.t()
    eg, eu = 2 * d * U * (xd.abs() @ gd.abs().t()), 2 * d * U * (xd.abs() @ ud.abs().t())
    near(gate, g, g.abs() * half(k) + eg + tiny(k), "gate")
    near(up, u, u.abs() * half(k) + eu + tiny(k), "up")
    a, da = act_reference(kind, g)
    want = a * u
    # |act'| <= 1.2; the exponential's argument is off by |g| u (gelu: its cubic by a few), some 16 u in all here
    tol = want.abs() * (half(k) + 8 * U) + (1.2 * eg + 16 * U * (g.abs() + g * g)) * (u.abs() + eu) + a.abs() * eu + tiny(k)
    near(out, want, tol, "out")
    if pad:
        for o in (out, gate, up):
            assert bool((o._base[:, off + f:] == 55).all()) and bool((o._base[:, :off] == 55).all())
    again = torch.empty(t, f, device="cuda", dtype=k)
    rt.gated_ffn(x, wg, wu, again, activation=kind)         # without the stored products: the same result
    if layout == "dense":
        assert torch.equal(again, out)


@pytest.mark.parametrize("out_ty", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["dense", "strided", "odd"])
@pytest.mark.parametrize("shape", FFN_SHAPES + [(40, 8200, 72)], ids=str)
def test_gated_ffn_int8(out_ty, shape, layout):
    t, d, f = shape
    k = TYPES[out_ty]
    g = torch.Generator().manual_seed(9)
    x, wg, wu = (torch.randint(-127, 128, s, generator=g).to(torch.int8) for s in ((t, d), (f, d), (f, d)))
    xs, gs, us = (0.5 + torch.rand(n, generator=g) for n in (t, f, f))
    gs, us, xs = gs * 0.02, us * 0.02, xs * 0.02 / d ** 0.5
    pad, off = {"strided": (16, 0), "odd": (3, 1)}.get(layout, (0, 0))
    out = strided(empty(t, f, ty=k), pad, off)
    rt.gated_ffn(strided(x.cuda(), pad, off), strided(wg.cuda(), pad, off), strided(wu.cuda(), pad, off), out,
                 scales=(xs.cuda(), gs.cuda(), us.cuda()))
    gg = (x.double() @ wg.double().t()) * xs.double()[:, None] * gs.double()
    uu = (x.double() @ wu.double().t()) * xs.double()[:, None] * us.double()
    a, _ = act_reference("silu", gg)
    # the sums are exact; a conversion and two products each, then as above
    want = a * uu
    near(out, want, want.abs() * (half(k) + 12 * U) + 1.2 * 20 * U * (gg.abs() + gg * gg) * uu.abs() + tiny(k), "out")


@pytest.mark.parametrize("layout", ["dense", "strided", "odd"])
@pytest.mark.parametrize("shape", FFN_SHAPES + [(1500, 40, 24)], ids=str)
@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_gated_ffn_backward(ty, shape, layout):
    t, d, f = shape
    k = TYPES[ty]
    kind = "gelu" if layout == "strided" else "silu"
    x, wg, wu = ffn_inputs(t, d, f, k)
    gate, up, dh = (dev(normal(j, t, f), k) for j in (5, 6, 7))
    pad, off = {"strided": (16, 0), "odd": (3, 1)}.get(layout, (0, 0))
    gx = strided(empty(t, d, ty=k), pad, off)
    gg, gu = (strided(empty(f, d, ty=k), pad, off) for _ in range(2))
    s = [strided(v, pad, off) for v in (dh, x, wg, wu, gate, up)]
    rt.gated_ffn_backward(*s, gx, gg, gu, activation=kind)
    a, da = act_reference(kind, f64(gate))
    dg, du = f64(dh) * f64(up) * da, f64(dh) * a
    # dg and du are rounded to the element type, after some 40 u of their factors (|gate| < 6)
    edg = dg.abs() * half(k) + 40 * U * (f64(dh) * f64(up)).abs() + tiny(k)
    edu = du.abs() * half(k) + 40 * U * f64(dh).abs() + tiny(k)
    xd, gd, ud = f64(x), f64(wg), f64(wu)
    want = dg @ gd + du @ ud
    sums = 4 * f * U * (dg.abs() @ gd.abs() + du.abs() @ ud.abs())
    near(gx, want, want.abs() * half(k) + 1.01 * (edg @ gd.abs() + edu @ ud.abs() + sums) + tiny(k), "grad_x")
    for got, p, ep, name in ((gg, dg, edg, "grad_w_gate"), (gu, du, edu, "grad_w_up")):
        want = p.t() @ xd
        near(got, want, want.abs() * half(k) + 1.01 * (ep.t() @ xd.abs() + 2 * t * U * (p.abs().t() @ xd.abs())) + tiny(k), name)
    if pad:
        for o, n in ((gx, d), (gg, d), (gu, d)):
            assert bool((o._base[:, off + n:] == 55).all()) and bool((o._base[:, :off] == 55).all())
    # one gradient at a time is the same gradient
    one = torch.empty(f, d, device="cuda", dtype=k)
    rt.gated_ffn_backward(*s, grad_w_up=one, activation=kind)
    assert torch.equal(one, gu)
    only = torch.empty(t, d, device="cuda", dtype=k)
    rt.gated_ffn_backward(*s, grad_x=only, activation=kind)
    assert torch.equal(only, gx)


def test_gated_ffn_gradients_are_the_slopes():
    t, d, f = 9, 40, 24
    x, wg, wu = ffn_inputs(t, d, f, torch.float16)
    dh = dev(normal(8, t, f), torch.float16)
    out, gate, up = (torch.empty(t, f, device="cuda", dtype=torch.float16) for _ in range(3))
    grads = [torch.empty_like(v) for v in (x, wg, wu)]
    e = 1e-5
    for kind in ("silu", "gelu"):
        rt.gated_ffn(x, wg, wu, out, activation=kind, gate=gate, up=up)
        rt.gated_ffn_backward(dh, x, wg, wu, gate, up, *grads, activation=kind)

        def total(x, wg, wu):
            return (act_reference(kind, x @ wg.t())[0] * (x @ wu.t()) * f64(dh)).sum()
        for i, v in enumerate((x, wg, wu)):
            step = normal(30 + i, *v.shape).double()
            args = [[f64(a) + (s * e * step if j == i else 0) for j, a in enumerate((x, wg, wu))] for s in (1, -1)]
            slope = (total(*args[0]) - total(*args[1])) / (2 * e)
            # each of the f (or t) terms of an element carries five roundings of half a step: gate, up, dg or du,
            # and the result; the derivatives are at most 1.2 and 0.6
            g, u = f64(x) @ f64(wg).t(), f64(x) @ f64(wu).t()
            size = f64(dh).abs() * (1 + g.abs()) * (1 + u.abs()) * 2
            per = {0: size @ (f64(wg).abs() + f64(wu).abs()), 1: size.t() @ f64(x).abs(), 2: size.t() @ f64(x).abs()}[i]
            assert abs(slope - (f64(grads[i]) * step).sum()) <= 5 * half(torch.float16) * (per * step.abs()).sum()


def test_gated_ffn_extreme_products():
    """Pre-activations far out on both sides: the activation's limits, no NaN from infinities inside."""
    x = torch.full((2, 8), 100.0, device="cuda", dtype=torch.bfloat16)
    x[1] = -100
    w = torch.full((8, 8), 50.0, device="cuda", dtype=torch.bfloat16)
    for kind in ("silu", "gelu"):
        out, gate, up = (torch.empty(2, 8, device="cuda", dtype=torch.bfloat16) for _ in range(3))
        rt.gated_ffn(x, w, w, out, activation=kind, gate=gate, up=up)
        assert bool((out[0] == 1.6e9).all() | ((out[0].double() / 1.6e9 - 1).abs() <= half(torch.bfloat16)).all())
        assert not bool(out[1].any())
        g = [torch.empty_like(v) for v in (x, w, w)]
        rt.gated_ffn_backward(torch.ones_like(out), x, w, w, gate, up, *g, activation=kind)
        assert all(bool(torch.isfinite(v).all()) for v in g)


def test_gated_ffn_without_tokens():
    d, f = 40, 24
    _, wg, wu = ffn_inputs(1, d, f, torch.bfloat16)
    x = torch.empty(0, d, device="cuda", dtype=torch.bfloat16)
    z = torch.empty(0, f, device="cuda", dtype=torch.bfloat16)
    rt.gated_ffn(x, wg, wu, z)
    gg, gu = empty(f, d, ty=torch.bfloat16), empty(f, d, ty=torch.bfloat16)
    rt.gated_ffn_backward(z, x, wg, wu, z, z, torch.empty_like(x), gg, gu)
    assert not bool(gg.any()) and not bool(gu.any())


# ---------------------------------------------------------------------------
# linear cross entropy
# ---------------------------------------------------------------------------
CE_SHAPES = [(1, 8, 1), (1, 64, 8), (1, 1024, 5000), (3, 1, 17), (2, 100, 1000), (16, 256, 777), (31, 136, 3001), (33, 65, 129),
             (64, 512, 2048), (129, 200, 1031), (257, 96, 512), (300, 264, 4099)]


def ce_inputs(t, d, v, ty, index=torch.int64):
    x = dev(normal(1, t, d), ty)
    w = dev(normal(2, v, d) * (2 / d ** 0.5), ty)
    targets = torch.randint(v, (t,), generator=torch.Generator().manual_seed(3)).to(index)
    if t > 4:
        targets[1], targets[t // 2], targets[2], targets[3] = -100, -1, v - 1, 0
    return x, w, targets.cuda()


@pytest.mark.parametrize("layout", ["dense", "strided", "odd"])
@pytest.mark.parametrize("shape", CE_SHAPES, ids=str)
@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_linear_cross_entropy(ty, shape, layout):
    t, d, v = shape
    x, w, targets = ce_inputs(t, d, v, TYPES[ty], torch.int32 if layout == "odd" else torch.int64)
    pad, off = {"strided": (16, 0), "odd": (3, 1)}.get(layout, (0, 0))
    loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
    rt.linear_cross_entropy(strided(x, pad, off), strided(w, pad, off), targets, loss, lse)
    z = f64(x) @ f64(w).t()
    ez = 2 * d * U * (f64(x).abs() @ f64(w).abs().t())
    want = torch.logsumexp(z, 1)
    # a logit's error moves lse by no more; the terms' exponentials are off by |z - max| u and a few u, the sum of
    # v terms joins at most v / 64 + 80 in a row
    tol = ez.amax(1) + ((z - z.amax(1, keepdim=True)).abs().amax(1) + v / 64 + 100 + want.abs()) * U
    near(lse, want, tol, "lse")
    live = targets.cpu() >= 0
    at = targets.cpu().long().clamp_min(0)
    want = torch.where(live, want - z.gather(1, at[:, None])[:, 0], 0.0)
    near(loss, want, tol + ez.amax(1) + want.abs() * U, "loss")
    assert not bool(loss.cpu()[~live].any())


@pytest.mark.parametrize("layout", ["dense", "strided", "odd"])
@pytest.mark.parametrize("shape", CE_SHAPES, ids=str)
@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_linear_cross_entropy_backward(ty, shape, layout):
    t, d, v = shape
    k = TYPES[ty]
    x, w, targets = ce_inputs(t, d, v, k, torch.int32 if layout == "odd" else torch.int64)
    g = dev(normal(4, t).abs() * 1e-3)
    if t > 6:
        g[5] = 0
    pad, off = {"strided": (16, 0), "odd": (3, 1)}.get(layout, (0, 0))
    xs, ws = strided(x, pad, off), strided(w, pad, off)
    z = f64(x) @ f64(w).t()
    lse = torch.logsumexp(z, 1)
    gx, gw = strided(empty(t, d, ty=k), pad, off), strided(empty(v, d, ty=k), pad, off)
    piece = {"dense": 0, "strided": 256, "odd": 200}[layout]
    rt.linear_cross_entropy_backward(xs, ws, targets, lse.float().cuda(), g, gx, gw, piece=piece)
    live = targets.cpu() >= 0
    gd = torch.where(live, f64(g), 0.0)[:, None]
    soft = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(z)
    hot[live, targets.cpu().long()[live]] = 1
    p = (soft - hot) * gd
    # p in fp32: z and lse are off by ez and half a step, the exponential by a few u; then one rounding to the element
    # type, fp16 at a scale where its smallest step is 2^-24 / 2^15 of the largest g
    ez = 2 * d * U * (f64(x).abs() @ f64(w).abs().t()) + (lse.abs()[:, None] + (z - lse[:, None]).abs() + 8) * U
    ep = soft * ez * gd + p.abs() * (half(k) + 8 * U) + gd * 4 * U + (2.0 ** -40 * f64(g).max() if ty == "f16" else 0.0)
    for got, want, e, name in ((gx, p @ f64(w), ep @ f64(w).abs() + 2 * v * U * (p.abs() @ f64(w).abs()), "grad_x"),
                               (gw, p.t() @ f64(x), ep.t() @ f64(x).abs() + 2 * t * U * (p.abs().t() @ f64(x).abs()), "grad_weight")):
        near(got, want, want.abs() * (half(k) + 4 * U) + 1.01 * e + tiny(k), name)
    if pad:
        for o in (gx, gw):
            assert bool((o._base[:, off + d:] == 55).all()) and bool((o._base[:, :off] == 55).all())
    assert not bool(gx[~live].any())
    only = torch.empty(v, d, device="cuda", dtype=k)
    rt.linear_cross_entropy_backward(xs, ws, targets, lse.float().cuda(), g, grad_weight=only, piece=piece)
    assert torch.equal(only, gw)
    only = torch.empty(t, d, device="cuda", dtype=k)
    rt.linear_cross_entropy_backward(xs, ws, targets, lse.float().cuda(), g, grad_x=only, piece=piece)
    assert torch.equal(only, gx)


def test_linear_cross_entropy_gradients_are_the_slopes():
    t, d, v = 11, 48, 300
    x, w, targets = ce_inputs(t, d, v, torch.float16)
    g = dev(normal(4, t).abs())
    loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
    gx, gw = torch.empty_like(x), torch.empty_like(w)
    rt.linear_cross_entropy(x, w, targets, loss, lse)
    rt.linear_cross_entropy_backward(x, w, targets, lse, g, gx, gw)
    live = targets.cpu() >= 0

    def total(x, w):
        z = x @ w.t()
        each = torch.logsumexp(z, 1) - z.gather(1, targets.cpu().clamp_min(0)[:, None])[:, 0]
        return (torch.where(live, each, 0.0) * f64(g)).sum()
    e = 1e-5
    for i, got in enumerate((gx, gw)):
        step = normal(40 + i, *got.shape).double()
        up, down = ([f64(a) + (s * e * step if j == i else 0) for j, a in enumerate((x, w))] for s in (1, -1))
        slope = (total(*up) - total(*down)) / (2 * e)
        # an element sums p times an operand: p's rounding and the result's own, each half a step
        p = torch.ones(t, v, dtype=torch.float64) * 2 / v
        p[live, targets.cpu()[live]] = 1
        p = p * f64(g)[:, None] * 4
        per = p @ f64(w).abs() if i == 0 else p.t() @ f64(x).abs()
        assert abs(slope - (f64(got) * step).sum()) <= 2 * half(torch.float16) * (per * step.abs()).sum()


@pytest.mark.parametrize("t", [1, 7, 150])
def test_linear_cross_entropy_rows_that_take_no_part(t):
    """All targets negative; targets past the vocabulary; infinite and NaN rows that are padding."""
    d, v = 64, 500
    x, w, targets = ce_inputs(t, d, v, torch.bfloat16)
    targets[:] = -100
    x[0] = float("nan")
    loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
    gx, gw = empty(t, d, ty=torch.bfloat16), empty(v, d, ty=torch.bfloat16)
    rt.linear_cross_entropy(x, w, targets, loss, lse)
    assert not bool(loss.any()) and bool(torch.isnan(lse[0])) and bool(torch.isfinite(lse[1:]).all())
    rt.linear_cross_entropy_backward(x, w, targets, lse, torch.ones(t, device="cuda"), gx, gw)
    assert not bool(gx.any()) and not bool(gw.any())
    x[0] = 1
    rt.linear_cross_entropy(x, w, targets, loss, lse)
    rt.linear_cross_entropy_backward(x, w, targets, lse, torch.ones(t, device="cuda"), gx, gw)
    assert not bool(gx.any()) and not bool(gw.any())
    targets[0] = v
    rt.linear_cross_entropy(x, w, targets, loss, lse)
    rt.linear_cross_entropy_backward(x, w, targets, lse, torch.ones(t, device="cuda"), gx, gw)
    assert bool(torch.isnan(loss[0])) and not bool(loss[1:].any()) and not bool(gx.any()) and not bool(gw.any())


@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [(40, 200, 300), (300, 263, 520)], ids=str)
def test_linear_cross_entropy_padding_holds_anything(ty, shape):
    """Padding rows of NaN with a huge or NaN grad_loss: the others' gradients are as without them."""
    t, d, v = shape
    k = TYPES[ty]
    x, w, targets = ce_inputs(t, d, v, k)
    pad = torch.arange(t, device="cuda") % 3 == 1
    targets = torch.where(pad, -100, targets.clamp_min(0))
    g = torch.where(pad, 0.0, dev(normal(4, t).abs() * 1e-3))
    results = []
    for dirty in (False, True):
        xs, gs = x.clone(), g.clone()
        if dirty:
            xs[pad], gs[pad] = float("nan"), 1e30
            gs[1] = float("nan")
        else:
            xs[pad] = 0
        loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
        gx, gw = torch.empty_like(x), torch.empty_like(w)
        rt.linear_cross_entropy(xs, w, targets, loss, lse)
        rt.linear_cross_entropy_backward(xs, w, targets, lse, gs, gx, gw)
        results.append((loss, gx, gw))
    for a, b in zip(*results):
        assert torch.equal(a, b) and bool(torch.isfinite(b).all())


def test_linear_cross_entropy_large_logits():
    """Logits of several thousand and equal logits: the maximum is taken out first."""
    t, d, v = 40, 32, 900
    x, w, targets = ce_inputs(t, d, v, torch.float16)
    x = x * 200
    x[7] = 0
    loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
    rt.linear_cross_entropy(x, w, targets, loss, lse)
    z = f64(x) @ f64(w).t()
    want = torch.logsumexp(z, 1)
    near(lse, want, 2 * d * U * (f64(x).abs() @ f64(w).abs().t()).amax(1) + (z.abs().amax(1) * 2 + 200) * U)
    gx, gw = torch.empty_like(x), torch.empty_like(w)
    rt.linear_cross_entropy_backward(x, w, targets, lse, torch.full((t,), 1e-6, device="cuda"), gx, gw)
    assert bool(torch.isfinite(gx).all()) and bool(torch.isfinite(gw).all())


def test_linear_cross_entropy_without_tokens():
    x = torch.empty(0, 64, device="cuda", dtype=torch.float16)
    w = dev(normal(1, 300, 64), torch.float16)
    none = torch.empty(0, device="cuda")
    rt.linear_cross_entropy(x, w, torch.empty(0, device="cuda", dtype=torch.int64), none, none)
    gw = empty(300, 64, ty=torch.float16)
    rt.linear_cross_entropy_backward(x, w, torch.empty(0, device="cuda", dtype=torch.int64), none, none, torch.empty_like(x), gw)
    assert not bool(gw.any())


# ---------------------------------------------------------------------------
# clipping by the global norm
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("sizes", [[1], [5], [16384], [16385, 1, 3], [0, 7, 0], [100003, 40000, 2], [9] * 130, [1_000_000, 3] * 3], ids=str)
@pytest.mark.parametrize("most", [0.0, 1.0, 1e9])
def test_clip_grad_norm(sizes, most):
    grads = [dev(normal(i, n) * 0.3, list(TYPES.values())[(i + len(sizes)) % 3]) for i, n in enumerate(sizes)]
    # every output lies between 9000 elements that stay as they are
    wide = [torch.full((g.numel() + 18000,), 55.0, device="cuda").to(g.dtype) for g in grads]
    outs, norm = [w[9000:9000 + g.numel()] for w, g in zip(wide, grads)], empty(1, ty=torch.float32)
    rt.clip_grad_norm(grads, outs, norm, most)
    for w, g in zip(wide, grads):
        assert bool((w[:9000] == 55).all()) and bool((w[9000 + g.numel():] == 55).all())
    want = sum(f64(g).square().sum() for g in grads).sqrt()
    near(norm, want.reshape(1), want * 4 * U)
    factor = min(1.0, most / (float(want) + 1e-6))
    for g, o in zip(grads, outs):
        near(o, f64(g) * factor, (f64(g) * factor).abs() * (half(g.dtype) + 8 * U) + tiny(g.dtype))
        if most == 1e9:
            assert torch.equal(g, o)                # nothing to clip: the same numbers
    rt.clip_grad_norm(grads, grads, norm, most)     # in place
    assert all(torch.equal(g, o) for g, o in zip(grads, outs))


def test_clip_grad_norm_values():
    """Squares beyond fp32, infinities, NaN, no tensors, unaligned tensors."""
    norm = empty(1, ty=torch.float32)
    big = torch.full((1000,), 1e30, device="cuda")
    out = torch.empty_like(big)
    rt.clip_grad_norm([big], [out], norm, 1.0)
    near(norm, torch.tensor([1e30 * 1000 ** 0.5], dtype=torch.float64), 1e32 * 4 * U)
    near(out, torch.full((1000,), 1000 ** -0.5, dtype=torch.float64), 8 * U)
    for value, check in ((float("inf"), lambda o: bool(torch.isnan(o[3])) and not bool(o[:3].any())),
                         (float("nan"), lambda o: bool(torch.isnan(o).all()))):
        g = torch.ones(1000, device="cuda", dtype=torch.float16)
        g[3] = value
        o = torch.empty_like(g)
        rt.clip_grad_norm([g], [o], norm, 1.0)
        assert not bool(torch.isfinite(norm[0])) and check(o)
    rt.clip_grad_norm([], [], norm, 1.0)
    assert float(norm[0]) == 0.0
    whole = dev(normal(1, 5000), torch.bfloat16)
    for off in (1, 3, 8):
        part, to = whole[off:off + 4000], torch.zeros(5000, device="cuda", dtype=torch.bfloat16)[off + 2:off + 4002]
        rt.clip_grad_norm([part], [to], norm, 0.5)
        factor = 0.5 / (float(f64(part).square().sum().sqrt()) + 1e-6)
        near(to, f64(part) * factor, (f64(part) * factor).abs() * (half(torch.bfloat16) + 8 * U))
        assert not bool(to._base[:off + 2].any()) and not bool(to._base[off + 4002:].any())


# ---------------------------------------------------------------------------
# repeated, side by side, together
# ---------------------------------------------------------------------------
def test_plans_repeat_bit_for_bit_and_alternate():
    """A plan launched again gives the same bits, also with another plan of the same operator, larger and with a
    workspace of its own, in between; nothing is kept from one call for the next."""
    def make(t, d, v, seed):
        x, w, targets = ce_inputs(t, d, v, torch.bfloat16)
        x = x + seed
        loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
        gx, gw = torch.empty_like(x), torch.empty_like(w)
        g = torch.full((t,), 1 / t, device="cuda")
        return ([rt.plan_linear_cross_entropy(x, w, targets, loss, lse),
                 rt.plan_linear_cross_entropy_backward(x, w, targets, lse, g, gx, gw, piece=512)], (loss, lse, gx, gw), x)
    (pa, oa, xa), (pb, ob, xb) = make(70, 200, 1500, 0), make(300, 264, 4099, 1)
    for p in pa:
        p.launch()
    first = [o.clone() for o in oa]
    for p in pb:
        p.launch()
    second = [o.clone() for o in ob]
    for _ in range(3):
        for one, two in zip(pb, pa):
            one.launch()
            two.launch()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, oa)) and all(torch.equal(a, b) for a, b in zip(second, ob))
    xa.neg_()                                   # new values in the same buffers are new inputs
    for p in pa:
        p.launch()
    want = torch.logsumexp(f64(xa) @ f64(pa[0].keep[1]).t(), 1)
    near(oa[1], want, 1e-4)
    assert not torch.equal(oa[2], first[2])


def test_two_queues_at_once():
    """Two contexts, each with its own queue and workspaces, launched in turn without waiting."""
    contexts = [rt.default_context(), rt.Context("hip:0")]
    t, d, f = 257, 264, 392
    x, wg, wu = ffn_inputs(t, d, f, torch.bfloat16)
    dh = dev(normal(8, t, f), torch.bfloat16)
    torch.cuda.synchronize()
    sets = []
    for ctx in contexts:
        out, gate, up = (torch.empty(t, f, device="cuda", dtype=torch.bfloat16) for _ in range(3))
        grads = [torch.empty_like(v) for v in (x, wg, wu)]
        plans = [rt.plan_gated_ffn(x, wg, wu, out, gate=gate, up=up),
                 rt.plan_gated_ffn_backward(dh, x, wg, wu, gate, up, *grads)]
        for p in plans:                         # the same launch on this context's queue
            p.args = (ctx.queue,) + p.args[1:]
        sets.append((plans, [out, gate, up] + grads))
    torch.cuda.synchronize()
    for _ in range(4):
        for k in range(2):
            for plans, _ in sets:
                plans[k].launch()
    for ctx in contexts:
        ctx.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(sets[0][1], sets[1][1]))


def test_a_training_step():
    """norm, feed-forward block, norm, loss, their backward passes and the clipping, one after the other as a program
    runs them, against the same in 64 bits."""
    t, d, v, k = 200, 136, 1000, torch.float16
    x, r = dev(normal(1, t, d), k), dev(normal(2, t, d), k)
    w1, w2 = dev(1 + 0.1 * normal(3, d)), dev(1 + 0.1 * normal(4, d))
    wg, wu, head = (dev(normal(s, n, d) * d ** -0.5, k) for s, n in ((5, d), (6, d), (7, v)))
    targets = torch.randint(v, (t,), generator=torch.Generator().manual_seed(8)).cuda()
    targets[::7] = -100
    live = (targets >= 0)
    g_loss = (live / live.sum() * 1024).float()             # scaled, as fp16 training does

    def e(*s, ty=k):
        return torch.empty(*s, device="cuda", dtype=ty)
    f32 = torch.float32
    h1, n1, r1, a, gate, up, h2, n2, r2 = e(t, d), e(t, d), e(t, ty=f32), e(t, d), e(t, d), e(t, d), e(t, d), e(t, d), e(t, ty=f32)
    loss, lse = e(t, ty=f32), e(t, ty=f32)
    gn2, ghead, gh2, gw2, gn1, gwg, gwu, gh1, gw1 = (e(t, d), e(v, d), e(t, d), e(d, ty=f32), e(t, d), e(d, d), e(d, d),
                                                     e(t, d), e(d, ty=f32))
    plans = [rt.plan_add_rms_norm(x, r, w1, n1, summed=h1, rstd=r1),
             rt.plan_gated_ffn(n1, wg, wu, a, gate=gate, up=up),
             rt.plan_add_rms_norm(a, h1, w2, n2, summed=h2, rstd=r2),
             rt.plan_linear_cross_entropy(n2, head, targets, loss, lse),
             rt.plan_linear_cross_entropy_backward(n2, head, targets, lse, g_loss, gn2, ghead),
             rt.plan_add_rms_norm_backward(gn2, h2, w2, r2, gh2, gw2),
             rt.plan_gated_ffn_backward(gh2, n1, wg, wu, gate, up, gn1, gwg, gwu),
             rt.plan_add_rms_norm_backward(gn1, h1, w1, r1, gh1, gw1, grad_summed=gh2)]
    grads = [ghead, gw2, gwg, gwu, gw1]
    norm, clipped = e(1, ty=f32), [torch.empty_like(g) for g in grads]
    plans.append(rt.plan_clip_grad_norm(grads, clipped, norm, 10.0))
    for _ in range(2):
        for p in plans:
            p.launch()
    torch.cuda.synchronize()
    leaves = [f64(q).requires_grad_() for q in (x, head, w2, wg, wu, w1)]
    xd, headd, w2d, wgd, wud, w1d = leaves

    def rms(h, w):
        return h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * w
    hd = xd + f64(r)
    nd = rms(hd, w1d)
    h2d = torch.nn.functional.silu(nd @ wgd.t()) * (nd @ wud.t()) + hd
    z = rms(h2d, w2d) @ headd.t()
    at = targets.cpu().clamp_min(0)[:, None]
    each = torch.where(live.cpu(), torch.logsumexp(z, 1) - z.gather(1, at)[:, 0], 0.0)
    (each * f64(g_loss)).sum().backward()
    # Along the way some sixteen tensors are rounded to fp16, each by at most half a step, and no stage
    # enlarges a relative error (in the 2-norm) by more than about two: 16 * 2 * 2^-11 = 2^-6.
    def off(got, want):
        return float((f64(got) - want.detach()).norm() / want.detach().norm())
    assert off(loss, each) < 2.0 ** -6
    wants = [headd.grad, w2d.grad, wgd.grad, wud.grad, w1d.grad]
    for got, want in zip([gh1] + grads, [xd.grad] + wants):
        assert off(got, want) < 2.0 ** -6
    total = sum(q.square().sum() for q in wants).sqrt()
    assert abs(float(norm[0]) / float(total) - 1) < 2.0 ** -6
    for got, want in zip(clipped, wants):
        assert off(got, want * min(1.0, 10.0 / float(total))) < 2.0 ** -5


def test_a_decoding_step_in_8_bits():
    """norm to 8 bits, weights quantised by the row kernel, the block on both."""
    t, d, f = 4, 4096, 520
    x, r = dev(normal(1, t, d), torch.float16), dev(normal(2, t, d), torch.float16)
    w = dev(1 + 0.1 * normal(3, d))
    weights = [dev(normal(s, f, d) * d ** -0.5, torch.float16) for s in (4, 5)]
    quantised = []
    for m in weights:
        q, s = torch.empty(f, d, device="cuda", dtype=torch.int8), empty(f, ty=torch.float32)
        rt.quantize_f16_i8(m, q, s)
        quantised.append((q, s))
    q, scale, h = torch.empty(t, d, device="cuda", dtype=torch.int8), empty(t, ty=torch.float32), torch.empty_like(x)
    out = empty(t, f, ty=torch.float16)
    rt.add_rms_norm(x, r, w, q, summed=h, scale=scale)
    rt.gated_ffn(q, quantised[0][0], quantised[1][0], out, scales=(scale, quantised[0][1], quantised[1][1]))
    xd = f64(q) * f64(scale)[:, None]
    g, u = (xd @ (f64(a) * f64(s)[:, None]).t() for a, s in quantised)
    a, _ = act_reference("silu", g)
    want = a * u
    near(out, want, want.abs() * (half(torch.float16) + 12 * U) + 1.2 * 20 * U * (g.abs() + g * g) * u.abs() + tiny(torch.float16))
    # and it stands for the block on the unquantised values: |x - q s| <= s / 2 on either side
    y = f64(h) / (f64(h).square().mean(1, keepdim=True) + 1e-6).sqrt() * f64(w)
    assert bool(((xd - y).abs() <= f64(scale)[:, None] * (0.5 + 1e-4)).all())


def test_refusals_on_the_device():
    """A refused call raises and launches nothing."""
    x = torch.ones(4, 16, device="cuda", dtype=torch.float16)
    out = empty(4, 16, ty=torch.float16)
    with pytest.raises(rt.HcRuntimeError, match="eps must not"):
        rt.add_rms_norm(x, None, None, out, eps=-1.0)
    p = rt.plan_linear_cross_entropy(x, x, torch.zeros(4, device="cuda", dtype=torch.int64), empty(4, ty=torch.float32),
                                     empty(4, ty=torch.float32))
    p.args = p.args[:-1] + (8,)
    with pytest.raises(rt.HcRuntimeError, match="workspace of 8 bytes"):
        p.launch(sync=True)
    torch.cuda.synchronize()
    assert bool((out == 77).all())


# ---------------------------------------------------------------------------
# every kernel of the products on the same shapes
# ---------------------------------------------------------------------------
@pytest.fixture(params=[1, 2, 3], ids=["general", "t128", "t256"])
def product_kernel(request):
    rt.set_variant("mma", request.param)
    yield request.param
    rt.set_variant("mma", 0)


# whole tiles; edges in every direction; k tiles of one, two, three and with every kind of tail (k is d forward, f
# and t backward)
TILED = [(1, 200, 264), (12, 328, 520), (100, 136, 136), (256, 64, 256), (512, 128, 512), (257, 200, 264), (300, 328, 391), (1000, 136, 520), (384, 1032, 777), (263, 256, 1001)]


@pytest.mark.parametrize("layout", ["dense", "strided"])
@pytest.mark.parametrize("shape", TILED, ids=str)
@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_block_on_every_kernel(product_kernel, ty, shape, layout):
    test_gated_ffn(ty, shape, layout)
    test_gated_ffn_backward(ty, shape, layout)


@pytest.mark.parametrize("shape", TILED, ids=str)
def test_block_int8_on_every_kernel(product_kernel, shape):
    t, d, f = shape
    test_gated_ffn_int8("bf16", (t, d // 16 * 16, f), "dense")
    test_gated_ffn_int8("f16", (t, d // 16 * 16, f), "strided")


@pytest.mark.parametrize("layout", ["dense", "strided", "odd"])
@pytest.mark.parametrize("shape", TILED, ids=str)
@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_cross_entropy_on_every_kernel(product_kernel, ty, shape, layout):
    test_linear_cross_entropy(ty, shape, layout)
    test_linear_cross_entropy_backward(ty, shape, layout)


def test_poisoned_surroundings(product_kernel):
    """NaN around every operand and output: nothing outside the windows is read into a result or written."""
    t, d, f, k = 300, 264, 520, torch.bfloat16

    def framed(x, pad=24):
        wide = torch.full((x.shape[0] + 2, x.shape[1] + pad), float("nan"), device="cuda", dtype=x.dtype)
        view = wide[1:-1, 8:8 + x.shape[1]]
        view.copy_(x)
        return view
    x, wg, wu = ffn_inputs(t, d, f, k)
    dh = dev(normal(8, t, f), k)
    plain, framed_out = [], []
    for wrap, results in ((lambda v: v, plain), (framed, framed_out)):
        out, gate, up = (wrap(empty(t, f, ty=k)) for _ in range(3))
        gx, gg, gu = wrap(empty(t, d, ty=k)), wrap(empty(f, d, ty=k)), wrap(empty(f, d, ty=k))
        xs, a, b, g = wrap(x), wrap(wg), wrap(wu), wrap(dh)
        rt.gated_ffn(xs, a, b, out, gate=gate, up=up)
        rt.gated_ffn_backward(g, xs, a, b, gate, up, gx, gg, gu)
        targets = (torch.arange(t) % f).cuda()
        loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
        cx, cw = wrap(empty(t, d, ty=k)), wrap(empty(f, d, ty=k))
        rt.linear_cross_entropy(xs, a, targets, loss, lse)
        rt.linear_cross_entropy_backward(xs, a, targets, lse, torch.ones(t, device="cuda"), cx, cw, piece=264)
        results += [out, gate, up, gx, gg, gu, loss, lse, cx, cw]
    for a, b in zip(plain, framed_out):
        assert torch.equal(a, b)
        if b._base is not None:
            inside = int(torch.isnan(b._base).sum())
            assert inside == b._base.numel() - b.numel()


# ---------------------------------------------------------------------------
# far offsets, graphs
# ---------------------------------------------------------------------------
def test_offsets_past_32_bits():
    """Rows more than 2^31 elements apart, and a weight matrix of more than 2^31 elements."""
    k = torch.bfloat16
    base = torch.zeros(3 * 1_100_000_000, device="cuda", dtype=k)
    far = base.as_strided((3, 520), (1_100_000_000, 1))
    x = dev(normal(1, 3, 520), k)
    far.copy_(x)
    y, q, scale = torch.empty_like(x), torch.empty(3, 520, device="cuda", dtype=torch.int8), empty(3, ty=torch.float32)
    rt.add_rms_norm(far, None, None, y)
    want = torch.empty_like(x)
    rt.add_rms_norm(x, None, None, want)
    assert torch.equal(y, want)
    rt.add_rms_norm(far, None, None, far)                    # results as far apart
    assert torch.equal(far, want)
    wg, wu = (dev(normal(s, 200, 520) * 0.04, k) for s in (2, 3))
    near_out, far_out = torch.empty(3, 200, device="cuda", dtype=k), base.as_strided((3, 200), (1_100_000_000, 1), 600)
    rt.gated_ffn(far, wg, wu, near_out)
    rt.gated_ffn(want, wg, wu, far_out)
    assert torch.equal(near_out, far_out)
    del base, far, far_out
    t, d, v = 256, 1024, 2_200_000
    w = torch.zeros(v, d, device="cuda", dtype=k)
    special = torch.tensor([0, 5, 1_000_003, 2_097_152, 2_097_153, 2_199_999], device="cuda")
    w[special] = dev(normal(4, 6, d) * 0.05, k)
    x = dev(normal(5, t, d), k)
    targets = special[torch.arange(t, device="cuda") % 6]
    loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
    rt.linear_cross_entropy(x, w, targets, loss, lse)
    z = f64(x) @ f64(w[special]).t()
    total = torch.exp(z).sum(1) + (v - 6)                    # every other logit is 0
    near(lse, total.log(), 1e-5)
    near(loss, total.log() - z[torch.arange(t), torch.arange(t) % 6], 2e-5)
    gx, gw = torch.empty_like(x), torch.empty_like(w)
    g = torch.full((t,), 1 / t, device="cuda")
    rt.linear_cross_entropy_backward(x, w, targets, lse, g, gx, gw)
    p = torch.exp(z) / total[:, None]
    p[torch.arange(t), torch.arange(t) % 6] -= 1
    p = p / t
    # p is rounded once (half a step; here it is up to 1 / t times the scale), the results once more
    want = p.t() @ f64(x)
    near(gw[special], want, want.abs() * half(k) + p.abs().t() @ f64(x).abs() * (half(k) + 2e-5))
    want = p @ f64(w[special])
    near(gx, want, want.abs() * half(k) + p.abs() @ f64(w[special]).abs() * (half(k) + 2e-5))
    rest = gw[torch.tensor([1, 1_500_000, 2_199_998], device="cuda")]
    want = ((1 / total / t)[:, None] * f64(x)).sum(0)
    near(rest, want.expand(3, d), want.abs() * half(k) + ((1 / total / t)[:, None] * f64(x).abs()).sum(0) * (half(k) + 2e-5))


def test_norm_backward_in_place():
    rows, cols = 600, 1032
    for t in TYPES.values():
        h, dy, ds = (dev(normal(k, rows, cols), t) for k in (1, 2, 3))
        w = dev(1 + 0.2 * normal(4, cols))
        rstd = (1 / (f64(h).square().mean(1) + 1e-6).sqrt()).float().cuda()
        want, gw = torch.empty_like(h), empty(cols, ty=torch.float32)
        rt.add_rms_norm_backward(dy, h, w, rstd, want, gw, grad_summed=ds)
        for which in (0, 1):
            a, b, g2 = dy.clone(), ds.clone(), empty(cols, ty=torch.float32)
            rt.add_rms_norm_backward(a, h, w, rstd, (a, b)[which], g2, grad_summed=b)
            assert torch.equal((a, b)[which], want) and torch.equal(gw, g2)


class Graph:
    """Launches of one queue recorded into a graph (the queue's second word is its stream)."""
    hip = None

    def __init__(self, ctx, launch):
        if Graph.hip is None:
            Graph.hip = C.CDLL("libamdhip64.so.7")       # the copy that is loaded already
        self.stream = C.c_void_p(C.cast(ctx.queue, C.POINTER(C.c_uint64))[1])
        graph, self.exec = C.c_void_p(), C.c_void_p()
        assert self.hip.hipStreamBeginCapture(self.stream, 1) == 0          # of this thread
        try:
            launch()
        finally:
            rc = self.hip.hipStreamEndCapture(self.stream, C.byref(graph))
        assert rc == 0 and self.hip.hipGraphInstantiate(C.byref(self.exec), graph, None, None, C.c_size_t(0)) == 0
        self.graph = graph

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exec, self.stream) == 0

    def close(self):
        assert self.hip.hipGraphExecDestroy(self.exec) == 0 and self.hip.hipGraphDestroy(self.graph) == 0


def test_captured_and_replayed():
    """Every operator recorded into graphs, two graphs of the same operators with plans of their own, replayed in turn
    with new inputs and eager work in between, against the eager results."""
    ctx = rt.default_context()
    k = torch.bfloat16

    def program(t, d, f, v):
        x, r = dev(normal(1, t, d), k), dev(normal(2, t, d), k)
        w1 = dev(1 + 0.1 * normal(3, d))
        wg, wu, head = (dev(normal(s, n, d) * d ** -0.5, k) for s, n in ((4, f), (5, f), (6, v)))
        targets = (torch.arange(t) % v).cuda()
        g = torch.full((t,), 1 / t, device="cuda")
        dh = dev(normal(7, t, f), k)
        h, n1, gx, gh, cx = (torch.empty_like(x) for _ in range(5))
        q, scale = torch.empty(t, d, device="cuda", dtype=torch.int8), empty(t, ty=torch.float32)
        out, gate, up = (torch.empty(t, f, device="cuda", dtype=k) for _ in range(3))
        gg, gu, gw, cw = torch.empty_like(wg), torch.empty_like(wu), empty(d, ty=torch.float32), torch.empty_like(head)
        rstd, loss, lse, norm = (empty(n, ty=torch.float32) for n in (t, t, t, 1))
        clipped = [torch.empty_like(a) for a in (gg, gu, gw, cw)]
        plans = [rt.plan_add_rms_norm(x, r, w1, n1, summed=h, rstd=rstd),
                 rt.plan_add_rms_norm(x, r, w1, q, scale=scale),
                 rt.plan_gated_ffn(n1, wg, wu, out, gate=gate, up=up),
                 rt.plan_gated_ffn_backward(dh, n1, wg, wu, gate, up, gx, gg, gu),
                 rt.plan_add_rms_norm_backward(gx, h, w1, rstd, gh, gw),
                 rt.plan_linear_cross_entropy(n1, head, targets, loss, lse),
                 rt.plan_linear_cross_entropy_backward(n1, head, targets, lse, g, cx, cw, piece=520),
                 rt.plan_clip_grad_norm([gg, gu, gw, cw], clipped, norm, 0.5)]
        return x, plans, [h, n1, q, scale, out, gate, up, gx, gg, gu, gh, gw, loss, lse, cx, cw, norm] + clipped

    programs = [program(20, 136, 200, 777), program(300, 264, 520, 1500)]
    for _, plans, _ in programs:
        for p in plans:
            p.launch()                                       # everything is loaded before the capture
    torch.cuda.synchronize()
    graphs = [Graph(ctx, lambda plans=plans: [p.launch() for p in plans]) for _, plans, _ in programs]
    for turn in range(4):
        wants = []
        for x, plans, outs in programs:
            x.copy_(dev(normal(50 + turn, *x.shape), k))
            torch.cuda.synchronize()
            for p in plans:
                p.launch()
            torch.cuda.synchronize()
            wants.append([o.clone() for o in outs])
            for o in outs:
                o.fill_(1)
        torch.cuda.synchronize()
        for gr in graphs:
            gr.replay()
        ctx.synchronize()
        for (_, _, outs), want in zip(programs, wants):
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), turn
    for gr in graphs:
        gr.close()


def test_nothing_is_allocated_by_a_launch():
    hip = C.CDLL("libamdhip64.so.7")

    def free_bytes():
        free, total = C.c_size_t(), C.c_size_t()
        assert hip.hipMemGetInfo(C.byref(free), C.byref(total)) == 0
        return free.value
    t, d, v = 200, 136, 1000
    x, w, targets = ce_inputs(t, d, v, torch.bfloat16)
    loss, lse, gx, gw = empty(t, ty=torch.float32), empty(t, ty=torch.float32), torch.empty_like(x), torch.empty_like(w)
    plans = [rt.plan_linear_cross_entropy(x, w, targets, loss, lse),
             rt.plan_linear_cross_entropy_backward(x, w, targets, lse, torch.ones(t, device="cuda"), gx, gw),
             rt.plan_add_rms_norm(x, None, None, gx)]
    for p in plans:
        p.launch(sync=True)
    before = free_bytes()
    for _ in range(5):
        for p in plans:
            p.launch(sync=True)
    assert free_bytes() == before


# ---------------------------------------------------------------------------
# many tokens with rows that are no multiple of 16 bytes: copied into the workspace
# ---------------------------------------------------------------------------
LAID = [(768, 9, 130), (801, 1003, 300), (1000, 63, 777), (1500, 530, 136), (2049, 1, 264)]


@pytest.mark.parametrize("layout", ["dense", "strided", "odd"])
@pytest.mark.parametrize("shape", LAID, ids=str)
@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_block_with_copied_rows(ty, shape, layout):
    assert rt.hcamdGatedFfnWorkspace(TYPES[ty] == torch.float16 and rt.F16 or rt.BF16, *shape) > 0
    test_gated_ffn(ty, shape, layout)
    test_gated_ffn_backward(ty, shape, layout)


@pytest.mark.parametrize("layout", ["dense", "strided", "odd"])
@pytest.mark.parametrize("shape", LAID + [(900, 1000, 200)], ids=str)
def test_block_int8_with_copied_rows(shape, layout):
    assert rt.hcamdGatedFfnWorkspace(rt.I8, *shape) > 0
    test_gated_ffn_int8("bf16", shape, layout)


# (the last two: several pieces of the weight in the forward pass, the last one of 4 and of 904 rows)
@pytest.mark.parametrize("layout", ["dense", "strided", "odd"])
@pytest.mark.parametrize("shape", LAID + [(900, 515, 60), (769, 16385, 4100), (770, 16401, 9096)], ids=str)
@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_cross_entropy_with_copied_rows(ty, shape, layout):
    test_linear_cross_entropy(ty, shape, layout)
    if shape[1] < 2000:
        test_linear_cross_entropy_backward(ty, shape, layout)


@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_cross_entropy_with_copied_rows_padding_holds_anything(ty):
    test_linear_cross_entropy_padding_holds_anything(ty, (800, 263, 520))


# ---------------------------------------------------------------------------
# dimensions shorter than a 16-byte piece, at more tokens than one pass over the weights takes
# ---------------------------------------------------------------------------
NARROW = [(64, 5, 40), (100, 7, 300), (200, 3, 9), (300, 64, 5), (300, 200, 1), (130, 137, 7), (40, 1, 1), (400, 11, 3), (133, 8, 8)]


@pytest.mark.parametrize("layout", ["dense", "strided", "odd"])
@pytest.mark.parametrize("shape", NARROW, ids=str)
@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_narrow_dimensions(ty, shape, layout):
    test_gated_ffn(ty, shape, layout)
    test_gated_ffn_backward(ty, shape, layout)
    test_gated_ffn_int8(ty, shape, layout)
    test_linear_cross_entropy(ty, shape, layout)
    test_linear_cross_entropy_backward(ty, shape, layout)


@pytest.mark.parametrize("t", [5, 40, 300, 800])
@pytest.mark.parametrize("d", [3, 9, 100, 517])
def test_operands_end_with_their_memory(t, d):
    """Operands whose last element is the last of its allocation, rows with NaN between them: nothing around a row
    changes a result."""
    f, k = 77, torch.bfloat16

    def last(x, pad):
        wide = torch.full((x.shape[0], x.shape[1] + pad), float("nan"), device="cuda", dtype=x.dtype)
        wide[:, pad:] = x
        return wide[:, pad:]
    x, wg, wu = ffn_inputs(t, d, f, k)
    dh = dev(normal(8, t, f), k)
    targets = (torch.arange(t) % f).cuda()
    results = []
    for pad in (0, 3):
        xs, a, b, g = (last(v, pad) for v in (x, wg, wu, dh))
        out, gate, up = (empty(t, f, ty=k) for _ in range(3))
        gx, gg, gu, cx, cw = empty(t, d, ty=k), empty(f, d, ty=k), empty(f, d, ty=k), empty(t, d, ty=k), empty(f, d, ty=k)
        rt.gated_ffn(xs, a, b, out, gate=gate, up=up)
        rt.gated_ffn_backward(g, xs, a, b, gate, up, gx, gg, gu)
        loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
        rt.linear_cross_entropy(xs, a, targets, loss, lse)
        rt.linear_cross_entropy_backward(xs, a, targets, lse, torch.ones(t, device="cuda"), cx, cw)
        results.append((out, gate, up, gx, gg, gu, loss, lse, cx, cw))
    # the two runs may take different kernels, which add in different orders: a stored value then differs by one step of
    # its type at most (2^-7), and a gradient made of stored gate, up, dg and du by as much again of the largest
    for p, q in zip(*results):
        assert bool(torch.isfinite(q).all()) and torch.allclose(p.float(), q.float(), rtol=2 ** -6, atol=2 ** -6 * float(p.abs().max()))


def test_copied_rows_captured_and_replayed():
    """The copies are part of the recorded work: new contents of the operands are seen by every replay."""
    ctx = rt.default_context()
    k, t, d, f = torch.bfloat16, 800, 131, 77
    x, wg, wu, dh = dev(normal(1, t, d), k), dev(normal(2, f, d), k), dev(normal(3, f, d), k), dev(normal(4, t, f), k)
    targets, g = (torch.arange(t) % f).cuda(), torch.full((t,), 1 / t, device="cuda")
    out, gate, up = (empty(t, f, ty=k) for _ in range(3))
    gx, gg, gu, cx, cw = empty(t, d, ty=k), empty(f, d, ty=k), empty(f, d, ty=k), empty(t, d, ty=k), empty(f, d, ty=k)
    loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
    outs = [out, gate, up, gx, gg, gu, loss, lse, cx, cw]
    plans = [rt.plan_gated_ffn(x, wg, wu, out, gate=gate, up=up),
             rt.plan_gated_ffn_backward(dh, x, wg, wu, gate, up, gx, gg, gu),
             rt.plan_linear_cross_entropy(x, wg, targets, loss, lse),
             rt.plan_linear_cross_entropy_backward(x, wg, targets, lse, g, cx, cw, piece=40)]
    for p in plans:
        p.launch(sync=True)
    graph = Graph(ctx, lambda: [p.launch() for p in plans])
    for turn in range(3):
        x.copy_(dev(normal(50 + turn, t, d), k))
        wg.copy_(dev(normal(60 + turn, f, d), k))
        torch.cuda.synchronize()
        for p in plans:
            p.launch(sync=True)
        want = [o.clone() for o in outs]
        for o in outs:
            o.fill_(1)
        torch.cuda.synchronize()
        graph.replay()
        ctx.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), turn
    graph.close()


def test_one_tensor_twice_is_refused():
    a, b, norm = torch.ones(8, device="cuda"), torch.ones(8, device="cuda"), empty(1, ty=torch.float32)
    for grads, outs in (([a, a], [a, a]), ([a, b], [b, a]), ([a, b], [a, a])):
        with pytest.raises(rt.HcRuntimeError, match="written twice"):
            rt.plan_clip_grad_norm(grads, outs, norm, 1.0)
    c = torch.empty_like(a)
    rt.clip_grad_norm([a, a], [c, torch.empty_like(a)], norm, 1.0)          # one gradient counted twice, two outputs
    assert torch.allclose(c, a / 4, rtol=1e-5)
    x = torch.ones(4, 16, device="cuda", dtype=torch.float16)
    with pytest.raises(rt.HcRuntimeError, match="two outputs are one buffer"):
        y = torch.empty_like(x)
        rt.add_rms_norm(x, None, None, y, summed=y)


# ---------------------------------------------------------------------------
# one pass over the weights for as many tokens as it takes
# ---------------------------------------------------------------------------
FEW = [(33, 64, 40), (48, 333, 97), (64, 136, 130), (65, 1001, 77), (100, 9, 300), (127, 264, 520), (128, 2000, 33), (90, 40, 1)]


@pytest.mark.parametrize("layout", ["dense", "strided", "odd"])
@pytest.mark.parametrize("shape", FEW, ids=str)
def test_up_to_128_tokens_in_one_pass(shape, layout):
    rt.set_variant("mma", 4)
    try:
        for ty in ("f16", "bf16"):
            test_gated_ffn(ty, shape, layout)
            test_linear_cross_entropy(ty, shape, layout)
            test_linear_cross_entropy_backward(ty, shape, layout)
            test_gated_ffn_int8(ty, shape, layout)
    finally:
        rt.set_variant("mma", 0)


@pytest.mark.parametrize("layout", ["dense", "odd"])
@pytest.mark.parametrize("shape", FEW + [(257, 200, 264), (300, 328, 391), (513, 640, 520)], ids=str)
def test_tiles_of_64_rows(shape, layout):
    rt.set_variant("mma", 5)
    try:
        for ty in ("f16", "bf16"):
            test_gated_ffn(ty, shape, layout)
            test_linear_cross_entropy(ty, shape, layout)
            test_linear_cross_entropy_backward(ty, shape, layout)
            test_gated_ffn_int8(ty, shape, layout)
    finally:
        rt.set_variant("mma", 0)


@pytest.mark.parametrize("layout", ["dense", "odd", "bare"])
@pytest.mark.parametrize("shape", [(3, 520), (700, 1016), (1030, 1000), (3, 2056), (600, 2057), (5, 4095), (520, 4096)], ids=str)
@pytest.mark.parametrize("ty", TYPES)
def test_row_kernels_on_both_sides_of_their_limits(ty, shape, layout):
    test_add_rms_norm(ty, shape, layout)
    test_add_rms_norm_int8(ty, shape, layout)
    test_add_rms_norm_backward(ty, shape, layout)
