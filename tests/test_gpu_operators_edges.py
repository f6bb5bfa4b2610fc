"""The language-model operators at the edges of their ranges, against their definitions in 64 bits:
values near the ends of a type, rows of zeros, dimensions past 32-bit offsets, calls without tokens.

Tolerances as in test_gpu_operators.py: U = 2^-24 for an fp32 operation, half(T) for a rounding to T,
tiny(T) for one among T's subnormal numbers."""
import numpy as np
import pytest

from hc_amd import runtime as rt

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_operators import Graph, TYPES, U, act_reference, dev, empty, f64, half, near, normal, strided, tiny  # noqa: E402


@pytest.mark.parametrize("d", [1, 5, 7, 8, 13, 200])
@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_cross_entropy_backward_without_tokens(ty, d):
    """No rows: the weight's gradient is zero, whatever the length of its rows (those shorter than 16 bytes are
    copied when there are rows)."""
    v, k = 300, TYPES[ty]
    none, targets = torch.empty(0, device="cuda"), torch.empty(0, device="cuda", dtype=torch.int64)
    x, w, gw = torch.empty(0, d, device="cuda", dtype=k), dev(normal(1, v, d), k), empty(v, d, ty=k)
    rt.linear_cross_entropy_backward(x, w, targets, none, none, torch.empty_like(x), gw)
    assert not bool(gw.any())
    rt.linear_cross_entropy_backward(x, w, targets, none, none, grad_x=torch.empty_like(x))


@pytest.mark.parametrize("d", [1, 5, 7, 8, 13, 200])
@pytest.mark.parametrize("ty", ["f16", "bf16"])
def test_gated_ffn_backward_without_tokens(ty, d):
    """No rows: the weights' gradients are zeros, whatever the length of their rows."""
    f, k = 40, TYPES[ty]
    x, z = torch.empty(0, d, device="cuda", dtype=k), torch.empty(0, f, device="cuda", dtype=k)
    w = dev(normal(1, f, d), k)
    gg, gu = empty(f, d, ty=k), empty(f, d, ty=k)
    rt.gated_ffn_backward(z, x, w, w, z, z, torch.empty_like(x), gg, gu)
    assert not bool(gg.any()) and not bool(gu.any())
    rt.gated_ffn_backward(z, x, w, w, z, z, grad_x=torch.empty_like(x))


def far_columns(n):
    """A few of n columns: both ends, and around the places where 32-bit byte offsets of 16-bit rows end."""
    at = [0, 1, 7, n // 3, n // 2 + 1, (1 << 22) - 1, 1 << 22, (1 << 22) + 5, n - 9, n - 8, n - 1]
    return torch.tensor(sorted({c for c in at if 0 <= c < n}))


# (the largest 16-bit rows whose 255th, 127th starts within 2^31 bytes hold 4.2 and 8.4 million values)
@pytest.mark.parametrize("shape", [(128, 128, 8_500_003), (256, 256, 4_300_000)], ids=str)
def test_block_backward_of_extreme_width(shape):
    """Pre-activation gradients whose rows lie more than 2^31 bytes apart in all: everything but a few columns is
    zero, so that the result is a short sum."""
    t, d, f = shape
    k = torch.bfloat16
    at = far_columns(f)
    n = len(at)
    vals = {name: dev(normal(i, t, n), k) for i, name in enumerate(("dh", "gate", "up"))}
    rows = {name: dev(normal(10 + i, n, d), k) for i, name in enumerate(("wg", "wu"))}
    x = dev(normal(20, t, d), k)
    dh, gate, up = (torch.zeros(t, f, device="cuda", dtype=k) for _ in range(3))
    wg, wu, gg, gu = (torch.zeros(f, d, device="cuda", dtype=k) for _ in range(4))
    for whole, name in ((dh, "dh"), (gate, "gate"), (up, "up")):
        whole[:, at.cuda()] = vals[name]
    wg[at.cuda()], wu[at.cuda()] = rows["wg"], rows["wu"]
    gx = empty(t, d, ty=k)
    rt.gated_ffn_backward(dh, x, wg, wu, gate, up, gx, gg, gu)
    a, da = act_reference("silu", f64(vals["gate"]))
    dg, du = f64(vals["dh"]) * f64(vals["up"]) * da, f64(vals["dh"]) * a
    edg = dg.abs() * half(k) + 40 * U * (f64(vals["dh"]) * f64(vals["up"])).abs() + tiny(k)
    edu = du.abs() * half(k) + 40 * U * f64(vals["dh"]).abs() + tiny(k)
    gd, ud, xd = f64(rows["wg"]), f64(rows["wu"]), f64(x)
    # (2 n + 2 terms that are not zero, and one addition each for at most 64 partial sums)
    want, sums = dg @ gd + du @ ud, (4 * n + 130) * U * (dg.abs() @ gd.abs() + du.abs() @ ud.abs())
    near(gx, want, want.abs() * half(k) + 1.01 * (edg @ gd.abs() + edu @ ud.abs() + sums) + tiny(k), "grad_x")
    for got, p, ep, name in ((gg, dg, edg, "grad_w_gate"), (gu, du, edu, "grad_w_up")):
        want = p.t() @ xd
        near(got[at.cuda()], want, want.abs() * half(k) + 1.01 * (ep.t() @ xd.abs() + 2 * t * U * (p.abs().t() @ xd.abs())) + tiny(k), name)
        got[at.cuda()] = 0
        assert not bool(got.any()), name


def test_cross_entropy_backward_of_an_extreme_piece():
    """One piece of the vocabulary whose rows of p lie more than 2^31 bytes apart in all; the weight is zero but for
    a few rows, so that dx is a short sum and every other row of dW is one and the same."""
    t, d, v = 128, 128, 8_500_003
    k = torch.bfloat16
    at = far_columns(v)
    n = len(at)
    x, rows = dev(normal(1, t, d), k), dev(normal(2, n, d) * 0.3, k)
    w, gw = torch.zeros(v, d, device="cuda", dtype=k), torch.full((v, d), 77.0, device="cuda", dtype=k)
    w[at.cuda()] = rows
    hit = torch.arange(t) % n
    targets = at[hit].cuda()
    loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
    rt.linear_cross_entropy(x, w, targets, loss, lse)
    z = f64(x) @ f64(rows).t()
    want_lse = (z.exp().sum(1) + (v - n)).log()
    # z is a sum of d products; an exponential's argument is off by a few u of itself on top
    ez = 2 * d * U * (f64(x).abs() @ f64(rows).abs().t()) + 16 * U * (z.abs() + want_lse[:, None])
    # a sum of v terms by tiles, of at most 32 additions each, joined by 64 lanes with v / 32 / 64 additions each
    share = ((z - want_lse[:, None]).exp() * ez).sum(1)
    near(lse, want_lse, 1.1 * share + (v / 2048 + 80) * U + want_lse.abs() * 4 * U, "lse")
    gx = empty(t, d, ty=k)
    grad = torch.full((t,), 1.0, device="cuda")
    rt.linear_cross_entropy_backward(x, w, targets, lse, grad, gx, gw, piece=v)
    p = (z - f64(lse)[:, None]).exp()
    ep = 1.1 * p * (ez + 8 * U)
    p[torch.arange(t), hit] -= 1
    ep += (p.abs() + ep) * half(k) + 2 * U + tiny(k)      # (the subtraction, the rounding to the type)
    rd, xd = f64(rows), f64(x)
    want = p @ rd
    near(gx, want, want.abs() * half(k) + 1.01 * (ep @ rd.abs() + (2 * n + 130) * U * (p.abs() @ rd.abs())) + tiny(k), "grad_x")
    want = p.t() @ xd
    near(gw[at.cuda()], want, want.abs() * half(k) + 1.01 * (ep.t() @ xd.abs() + 2 * t * U * (p.abs().t() @ xd.abs())) + tiny(k), "grad_weight")
    other = torch.ones(v, dtype=torch.bool)
    other[at] = False
    first = gw[2]
    assert bool((gw[other.cuda()] == first).all())
    p0 = (-f64(lse)).exp()
    want = p0 @ xd
    near(first, want, want.abs() * half(k) + 1.01 * ((p0 * (half(k) + 300 * U)) @ xd.abs()) + tiny(k), "the other rows")


@pytest.mark.parametrize("layout", ["dense", "odd"])
@pytest.mark.parametrize("size", [1e-6, 1e-4, 3e4])
@pytest.mark.parametrize("shape", [(5, 40, 24), (129, 65, 77), (512, 256, 512), (700, 520, 640)], ids=str)
def test_block_backward_gradients_at_the_ends_of_fp16(shape, size, layout):
    """Gradients whose products with the activations leave fp16's normal numbers on either side: dg and du keep their
    relative precision, and nothing becomes infinite that the results can hold."""
    t, d, f = shape
    k = torch.float16
    kind = "gelu" if layout == "odd" else "silu"
    by = 0.01 if size > 1 else 1.0                      # (results of large gradients stay below 65504)
    x, wg, wu = dev(normal(1, t, d) * by, k), dev(normal(2, f, d) * by * d ** -0.5, k), dev(normal(3, f, d) * by * d ** -0.5, k)
    gate, up = dev(normal(5, t, f), k), dev(normal(6, t, f), k)
    dh = dev((normal(7, t, f) * size).clamp(-6e4, 6e4), k)
    pad, off = (3, 1) if layout == "odd" else (0, 0)
    gx = strided(empty(t, d, ty=k), pad, off)
    gg, gu = (strided(empty(f, d, ty=k), pad, off) for _ in range(2))
    rt.gated_ffn_backward(*[strided(v, pad, off) for v in (dh, x, wg, wu, gate, up)], gx, gg, gu, activation=kind)
    a, da = act_reference(kind, f64(gate))
    dg, du = f64(dh) * f64(up) * da, f64(dh) * a
    # the largest of them is scaled to 2^14 at least: half a subnormal step is then that part of it
    low = tiny(k) * 2.0 ** -14 * max(dg.abs().max(), du.abs().max())
    edg = dg.abs() * half(k) + 40 * U * (f64(dh) * f64(up)).abs() + low
    edu = du.abs() * half(k) + 40 * U * f64(dh).abs() + low
    xd, gd, ud = f64(x), f64(wg), f64(wu)
    want = dg @ gd + du @ ud
    assert want.abs().max() < 65000
    sums = 4 * f * U * (dg.abs() @ gd.abs() + du.abs() @ ud.abs())
    near(gx, want, want.abs() * half(k) + 1.01 * (edg @ gd.abs() + edu @ ud.abs() + sums) + tiny(k), "grad_x")
    for got, p, ep, name in ((gg, dg, edg, "grad_w_gate"), (gu, du, edu, "grad_w_up")):
        want = p.t() @ xd
        assert want.abs().max() < 65000
        near(got, want, want.abs() * half(k) + 1.01 * (ep.t() @ xd.abs() + 2 * t * U * (p.abs().t() @ xd.abs())) + tiny(k), name)


def test_block_backward_fp16_that_is_zero_or_not_finite():
    """Gradients that are all zero; one that is infinite or NaN reaches its own row and column only."""
    t, d, f = 40, 64, 96
    k = torch.float16
    x, w = dev(normal(1, t, d), k), dev(normal(2, f, d) * 0.1, k)
    gate, up = dev(normal(3, t, f), k), dev(normal(4, t, f), k)
    for bad in (0.0, float("inf"), float("nan")):
        dh = torch.zeros(t, f, device="cuda", dtype=k)
        dh[5, 7] = bad
        gx, gg, gu = (torch.full_like(v, 77.0) for v in (x, w, w))
        rt.gated_ffn_backward(dh, x, w, w, gate, up, gx, gg, gu)
        for o, row in ((gx, 5), (gg, 7), (gu, 7)):
            assert bool(torch.isfinite(o[row]).any()) == (bad == 0.0)
            o[row] = 0
            assert not bool(o.any())


@pytest.mark.parametrize("cols", [1, 100, 4096, 20000])
@pytest.mark.parametrize("ty", TYPES)
def test_a_row_of_zeros_has_scale_0_without_eps(ty, cols):
    x = dev(normal(1, 4, cols), TYPES[ty])
    x[1] = 0
    w = torch.ones(cols, device="cuda")
    for weight, zeros in ((w, [1]), (w * 0, [0, 1, 2, 3])):
        q, scale = torch.full((4, cols), 55, device="cuda", dtype=torch.int8), empty(4, ty=torch.float32)
        rt.add_rms_norm(x, None, weight, q, eps=0.0, scale=scale)
        assert [r for r in range(4) if float(scale[r]) == 0.0] == zeros, scale
        assert not bool(q[zeros].any()) and bool(torch.isfinite(scale).all())


@pytest.mark.parametrize("most", [1.0, 1e30])
@pytest.mark.parametrize("size", [1e18, 1e37, 3e38])
@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_clip_of_gradients_whose_norm_leaves_fp32(ty, size, most):
    """Finite gradients are scaled to the norm asked for, also where their norm is beyond fp32 or the factor below its
    normal numbers.  The factor is off by 3 u (64 bits, rounded once), the product by one more."""
    k = TYPES[ty]
    g = [dev(torch.full((n,), size) * (1 - 0.5 * torch.rand(n, generator=torch.Generator().manual_seed(n))), k) for n in (100, 4099, 3)]
    g.append(dev(torch.tensor([1.0, 1e-30, 0.0]), torch.float32))
    out, norm = [torch.empty_like(v) for v in g], empty(1, ty=torch.float32)
    rt.clip_grad_norm(g, out, norm, most)
    total = float(sum(f64(v).square().sum() for v in g).sqrt())
    if total < 3e38:
        near(norm, torch.tensor([total], dtype=torch.float64), 2 * total * U)
    else:
        assert bool(torch.isinf(norm).all())
    for v, o in zip(g, out):
        want = f64(v) * min(1.0, most / (total + 1e-6))
        near(o, want, want.abs() * (4 * U + (half(k) if v.dtype == k else 0)) + tiny(torch.float32), "clipped")


def test_a_workspace_outlives_the_kernels_that_use_it(monkeypatch):
    """sync=False of a call that brings a workspace of its own waits all the same; one without does not."""
    events = []

    class Watched(rt.DeviceArray):
        def free(self):
            if getattr(self, "ptr", None):
                events.append("free")
            super().free()

    monkeypatch.setattr(rt, "_workspace", lambda n, ctx: Watched((n,), np.uint8, ctx) if n else None)
    inner = rt.Context.synchronize
    monkeypatch.setattr(rt.Context, "synchronize", lambda self: (events.append("wait"), inner(self))[1])
    k = torch.float16
    for (t, d, f), want in (((800, 33, 40), ["wait", "free"]), ((3, 5, 16), ["wait", "free"]), ((3, 64, 16), [])):
        x, wg, wu = dev(normal(1, t, d), k), dev(normal(2, f, d), k), dev(normal(3, f, d), k)
        out = empty(t, f, ty=k)
        torch.cuda.synchronize()
        events.clear()
        rt.gated_ffn(x, wg, wu, out, sync=False)
        assert events == want, (t, d, f)
        rt.default_context().synchronize()
        a, _ = act_reference("silu", f64(x) @ f64(wg).t())
        want_out = a * (f64(x) @ f64(wu).t())
        assert float((f64(out) - want_out).norm() / want_out.norm()) < 4 * half(k)


def test_results_are_rounded_alike_with_and_without_partial_sums():
    """The loss's gradients are fp32 values before they are rounded to the type, also those that partial sums are
    folded into.  With a weight of zeros every p is one 16-bit value, and the rows of x are such that the sums of
    a column are its own number: the result is known to the bit."""
    t, d, v = 4096, 1024, 1000
    k = torch.float16
    w = torch.zeros(v, d, device="cuda", dtype=k)
    targets = torch.zeros(t, device="cuda", dtype=torch.int64)
    lse = torch.full((t,), float(np.log(np.float32(v))), device="cuda")
    gw = torch.empty_like(w)
    x = torch.zeros(t, d, dtype=k)
    for bit in range(10):                               # in different parts of the sum over the tokens
        x[bit * 400] = (torch.arange(d) >> bit & 1) * 2.0 ** bit
    x = x.cuda()
    # p in 16 bits, from a gradient that nothing has to be undone for but a power of two
    rt.linear_cross_entropy_backward(x, w, targets, lse, torch.ones(t, device="cuda"), None, gw)
    p = float(f64(gw[1, 1])) * 2.0 ** 15
    assert p == float(np.float16(p)) and 30 < p < 35
    sums = p * np.arange(d)                             # 21 bits: exact in fp32 and as sums
    # gradients for which rounding in one step and in two differ somewhere, both known exactly in 64 bits
    tried = np.random.default_rng(1).uniform(0.01, 5, 4000).astype(np.float32)
    once = sums * (tried / np.float32(2.0 ** 15)).astype(np.float64)[:, None]
    twice = once.astype(np.float32).astype(np.float16)
    chosen = np.flatnonzero((once.astype(np.float16) != twice).any(1))[:8]
    assert len(chosen) == 8
    for i in chosen:
        rt.linear_cross_entropy_backward(x, w, targets, lse, torch.full((t,), float(tried[i]), device="cuda"), None, gw)
        assert np.array_equal(gw[1].cpu().numpy(), twice[i]), tried[i]


@pytest.mark.parametrize("t", [1, 20, 100, 300])
def test_loss_of_infinite_logits(t):
    """An infinite logit: the log-sum-exp is infinite (or, all being -infinity, minus that), not NaN."""
    d, v, k = 64, 1031, torch.bfloat16
    x, w = torch.zeros(t, d, device="cuda", dtype=k), torch.zeros(v, d, device="cuda", dtype=k)
    x[:, 0], x[:, 1] = 3e38, 1
    w[:, 1] = dev(normal(1, v), k)
    w[777, 0] = 3e38                                    # column 777: +infinity
    targets = torch.zeros(t, device="cuda", dtype=torch.int64)
    loss, lse = empty(t, ty=torch.float32), empty(t, ty=torch.float32)
    rt.linear_cross_entropy(x, w, targets, loss, lse)
    assert bool((lse == float("inf")).all()) and bool((loss == float("inf")).all()), (lse[:3], loss[:3])
    w[777, 0] = -3e38                                   # -infinity: its term is 0
    rt.linear_cross_entropy(x, w, targets, loss, lse)
    z = f64(x[:1, 1:]) @ f64(w[:, 1:]).t()
    z[0, 777] = -float("inf")
    want = torch.logsumexp(z, 1).expand(t)
    near(lse, want, 200 * U * want.abs(), "lse")
    near(loss, want - z[0, 0], 200 * U * (want.abs() + z[0, 0].abs()), "loss")


@pytest.mark.parametrize("shape", [(1, 64, 40), (33, 333, 97), (130, 129, 200), (300, 1024, 257), (513, 640, 520), (800, 33, 40)], ids=str)
def test_gated_ffn_int8_gelu(shape):
    t, d, f = shape
    k = torch.bfloat16
    g = torch.Generator().manual_seed(9)
    x, wg, wu = (torch.randint(-127, 128, s, generator=g).to(torch.int8) for s in ((t, d), (f, d), (f, d)))
    xs, gs, us = (0.5 + torch.rand(n, generator=g) for n in (t, f, f))
    gs, us, xs = gs * 0.02, us * 0.02, xs * 0.02 / d ** 0.5
    out = empty(t, f, ty=k)
    rt.gated_ffn(x.cuda(), wg.cuda(), wu.cuda(), out, activation="gelu", scales=(xs.cuda(), gs.cuda(), us.cuda()))
    gg = (x.double() @ wg.double().t()) * xs.double()[:, None] * gs.double()
    uu = (x.double() @ wu.double().t()) * xs.double()[:, None] * us.double()
    a, _ = act_reference("gelu", gg)
    # the sums are exact; a conversion and two products each; the exponential's argument, 1.6 (g + 0.045 g^3), is
    # off by some 8 u of itself
    want = a * uu
    near(out, want, want.abs() * (half(k) + 12 * U) + 24 * U * (gg.abs() + gg * gg + 0.08 * gg ** 4) * uu.abs() + tiny(k), "out")


def test_fp16_block_backward_captured_and_replayed():
    """The scaling follows the gradients of each replay: two graphs with plans of their own, gradients of other sizes
    every time and eager work in between, against the eager results."""
    ctx, k = rt.default_context(), torch.float16

    def program(t, d, f):
        x, gate, up, dh = dev(normal(1, t, d) * 0.01, k), dev(normal(2, t, f), k), dev(normal(3, t, f), k), empty(t, f, ty=k)
        w = [dev(normal(s, f, d) * 0.01 * d ** -0.5, k) for s in (4, 5)]
        outs = [torch.empty_like(v) for v in (x, *w)]
        return dh, rt.plan_gated_ffn_backward(dh, x, *w, gate, up, *outs), outs

    programs = [program(20, 136, 200), program(801, 131, 260)]
    for dh, plan, _ in programs:
        plan.launch(sync=True)                          # everything is loaded before the capture
    graphs = [Graph(ctx, plan.launch) for _, plan, _ in programs]
    for turn, size in enumerate((1.0, 1e-6, 1e4, 0.0, 1e-3)):
        wants = []
        for dh, plan, outs in programs:
            dh.copy_(dev(normal(50 + turn, *dh.shape) * size, k))
            torch.cuda.synchronize()
            plan.launch(sync=True)
            wants.append([o.clone() for o in outs])
            assert all(bool(torch.isfinite(o).all()) and bool(o.any()) == (size > 0) for o in outs), size
            for o in outs:
                o.fill_(1)
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        ctx.synchronize()
        for (_, _, outs), want in zip(programs, wants):
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), size
    for graph in graphs:
        graph.close()
