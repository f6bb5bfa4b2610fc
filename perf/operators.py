"""The language-model operators of hc_amd.runtime as measured cases.

Four operators, each with the other direction where it has one:

  norm   h = x + residual in the storage type, y = h / rms(h) * weight; y in the
         storage type (with its backward pass) or in 8 bits with a scale a row
  ffn    act(x Wg') * (x Wu'): the gated half of a feed-forward block, from
         16-bit operands (with its backward pass) or 8-bit ones with scales
  ce     softmax cross entropy of x W' against targets, rows of loss and
         log-sum-exp, the logits never stored (with the gradients of x and W)
  clip   global norm of many gradient tensors, and the clipped tensors

`own` false: the plain form in elementary torch operations, 32 bits throughout
and one rounding at the end; true: the framework's kernels, launched through the
plans that a program builds once and keeps."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
EPS = 1e-6
MAX_NORM = 1.0


def listed():
    return [
        # a decoding step of four sequences: the 8-bit activations of the next product; latency
        {"name": "norm int8 4x4096", "op": "norm", "mode": "int8", "rows": 4, "cols": 4096, "type": "bf16"},
        # a training step's norm over 8192 tokens, both directions
        {"name": "norm train 8192x4096", "op": "norm", "mode": "train", "rows": 8192, "cols": 4096, "type": "bf16"},
        # a long prompt in the shape of the row-quantisation benchmark
        {"name": "norm int8 16384x4096", "op": "norm", "mode": "int8", "rows": 16384, "cols": 4096, "type": "f16"},
        # single-token decoding: two weight matrices read once
        {"name": "ffn decode 1", "op": "ffn", "mode": "forward", "tokens": 1, "d": 4096, "f": 11264, "type": "bf16"},
        # a prompt of 2000 tokens through 8-bit weights
        {"name": "ffn int8 2000", "op": "ffn", "mode": "forward", "tokens": 2000, "d": 4096, "f": 11264, "type": "i8"},
        # a training step: the forward pass and all three gradients
        {"name": "ffn train 4096", "op": "ffn", "mode": "train", "tokens": 4096, "d": 4096, "f": 11264, "type": "bf16"},
        # a small model with odd sizes, both directions
        {"name": "ffn train odd", "op": "ffn", "mode": "train", "tokens": 333, "d": 1001, "f": 2731, "type": "f16"},
        # scoring a short continuation: the loss alone
        {"name": "ce score 32", "op": "ce", "mode": "forward", "tokens": 32, "d": 4096, "vocab": 32000, "type": "bf16"},
        # a training step of a small model with an odd vocabulary
        {"name": "ce train odd", "op": "ce", "mode": "train", "tokens": 1000, "d": 1024, "vocab": 50021, "type": "f16"},
        # a training step over a large vocabulary
        {"name": "ce train 4096x131072", "op": "ce", "mode": "train", "tokens": 4096, "d": 4096, "vocab": 131072,
         "type": "bf16"},
        # the gradients of an adapter: a dozen small tensors; latency
        {"name": "clip 12 small", "op": "clip", "count": 12, "elems": 200_000, "type": "f32"},
        # the gradients of a model of 400 million weights
        {"name": "clip 60 large", "op": "clip", "count": 60, "elems": 400_000_000, "type": "bf16"},
    ]


def draw(rng):
    def size(lo, hi):  # spread over the logarithm
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    op = rng.choice(["norm", "ffn", "ce", "clip"])
    if op == "norm":
        return {"op": op, "mode": rng.choice(["int8", "train"]), "rows": size(1, 16384), "cols": size(64, 16384),
                "type": rng.choice(["bf16", "f16", "f32"])}
    if op == "ffn":
        kind = rng.choice(["bf16", "f16", "i8"])
        return {"op": op, "mode": "forward" if kind == "i8" else rng.choice(["forward", "train"]),
                "tokens": size(1, 4096), "d": size(64, 4096), "f": size(64, 11264), "type": kind}
    if op == "ce":
        return {"op": op, "mode": rng.choice(["forward", "train"]), "tokens": size(1, 4096), "d": size(64, 4096),
                "vocab": size(1000, 131072), "type": rng.choice(["bf16", "f16"])}
    return {"op": op, "count": size(1, 60), "elems": size(10_000, 200_000_000),
            "type": rng.choice(["bf16", "f16", "f32"])}


def tensor_sizes(case):
    """Element counts of the clipped tensors: a few large ones, many small and odd ones."""
    n, share = case["count"], [1.0 / (1 + i) for i in range(case["count"])]
    return [max(1, int(case["elems"] * s / sum(share))) for s in share][:n]


def prepare(case, seed):
    """Inputs from the seed; with `own`, the result buffers and launch plans that a program keeps beside them."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    s = {"case": case}
    if case["op"] == "norm":
        r, c, ty = case["rows"], case["cols"], TYPES[case["type"]]
        # the residual stream has a few channels far larger than the rest
        big = torch.where(torch.rand(c, device="cuda", generator=gen) < 0.01, 20.0, 1.0)
        s["x"] = normal(r, c).to(ty)
        s["residual"] = (normal(r, c) * big).to(ty)
        s["weight"] = 1 + 0.1 * normal(c)
        if case["mode"] == "train":
            s["grad_out"], s["grad_summed"] = normal(r, c).to(ty), normal(r, c).to(ty)
    elif case["op"] == "ffn":
        t, d, f, ty = case["tokens"], case["d"], case["f"], TYPES[case["type"]]
        if ty == torch.int8:
            def bits(*shape):
                return (normal(*shape) * 32).round().clamp(-127, 127).to(torch.int8)
            s["x"], s["w_gate"], s["w_up"] = bits(t, d), bits(f, d), bits(f, d)
            s["x_scale"] = (0.02 + 0.02 * torch.rand(t, device="cuda", generator=gen))
            s["gate_scale"] = (0.5 + torch.rand(f, device="cuda", generator=gen)) * (0.04 / math.sqrt(d))
            s["up_scale"] = (0.5 + torch.rand(f, device="cuda", generator=gen)) * (0.04 / math.sqrt(d))
        else:
            s["x"] = normal(t, d).to(ty)
            s["w_gate"], s["w_up"] = ((normal(f, d) / math.sqrt(d)).to(ty) for _ in range(2))
            if case["mode"] == "train":
                s["grad_out"] = normal(t, f).to(ty)
    elif case["op"] == "ce":
        t, d, v, ty = case["tokens"], case["d"], case["vocab"], TYPES[case["type"]]
        s["x"] = normal(t, d).to(ty)
        s["weight"] = (normal(v, d) * (2 / math.sqrt(d))).to(ty)
        s["targets"] = torch.randint(v, (t,), device="cuda", generator=gen)
        if t > 1:  # padding and prompts take no part
            s["targets"][torch.rand(t, device="cuda", generator=gen) < 0.05] = -100
        if case["mode"] == "train":
            live = s["targets"] >= 0
            s["grad_loss"] = live.float() / live.sum().clamp_min(1)
    else:
        ty = TYPES[case["type"]]
        s["grads"] = [(normal(n) * 0.01).to(ty) for n in tensor_sizes(case)]
    if own:
        keep_plans(case, s)
    return s


def keep_plans(case, s):
    import hc_amd.runtime as rt

    def empty(*shape, dtype):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    ty = TYPES[case["type"]]
    if case["op"] == "norm":
        x, r, c = s["x"], case["rows"], case["cols"]
        h = torch.empty_like(x)
        if case["mode"] == "int8":
            q, scale = empty(r, c, dtype=torch.int8), empty(r, dtype=torch.float32)
            s["plans"] = [rt.plan_add_rms_norm(x, s["residual"], s["weight"], q, eps=EPS, summed=h, scale=scale)]
            s["outputs"] = [h, q, scale]
        else:
            y, rstd = torch.empty_like(x), empty(r, dtype=torch.float32)
            gx, gw = torch.empty_like(x), empty(c, dtype=torch.float32)
            s["plans"] = [rt.plan_add_rms_norm(x, s["residual"], s["weight"], y, eps=EPS, summed=h, rstd=rstd),
                          rt.plan_add_rms_norm_backward(s["grad_out"], h, s["weight"], rstd, gx, gw,
                                                        grad_summed=s["grad_summed"])]
            s["outputs"] = [h, y, gx, gw]
    elif case["op"] == "ffn":
        t, f = case["tokens"], case["f"]
        if ty == torch.int8:
            out = empty(t, f, dtype=torch.bfloat16)
            s["plans"] = [rt.plan_gated_ffn(s["x"], s["w_gate"], s["w_up"], out,
                                            scales=(s["x_scale"], s["gate_scale"], s["up_scale"]))]
            s["outputs"] = [out]
        elif case["mode"] == "forward":
            out = empty(t, f, dtype=ty)
            s["plans"] = [rt.plan_gated_ffn(s["x"], s["w_gate"], s["w_up"], out)]
            s["outputs"] = [out]
        else:
            out, gate, up = (empty(t, f, dtype=ty) for _ in range(3))
            gx, gwg, gwu = torch.empty_like(s["x"]), torch.empty_like(s["w_gate"]), torch.empty_like(s["w_up"])
            s["plans"] = [rt.plan_gated_ffn(s["x"], s["w_gate"], s["w_up"], out, gate=gate, up=up),
                          rt.plan_gated_ffn_backward(s["grad_out"], s["x"], s["w_gate"], s["w_up"], gate, up,
                                                     gx, gwg, gwu)]
            s["outputs"] = [out, gx, gwg, gwu]
    elif case["op"] == "ce":
        t = case["tokens"]
        loss, lse = empty(t, dtype=torch.float32), empty(t, dtype=torch.float32)
        s["plans"] = [rt.plan_linear_cross_entropy(s["x"], s["weight"], s["targets"], loss, lse)]
        s["outputs"] = [loss, lse]
        if case["mode"] == "train":
            gx, gw = torch.empty_like(s["x"]), torch.empty_like(s["weight"])
            s["plans"].append(rt.plan_linear_cross_entropy_backward(s["x"], s["weight"], s["targets"], lse,
                                                                    s["grad_loss"], gx, gw))
            s["outputs"] += [gx, gw]
    else:
        outs, norm = [torch.empty_like(g) for g in s["grads"]], empty(1, dtype=torch.float32)
        s["plans"] = [rt.plan_clip_grad_norm(s["grads"], outs, norm, MAX_NORM)]
        s["outputs"] = [norm] + outs


def run(s):
    if own:
        for plan in s["plans"]:
            plan.launch()
        return s["outputs"]
    return {"norm": plain_norm, "ffn": plain_ffn, "ce": plain_ce, "clip": plain_clip}[s["case"]["op"]](s)


def plain_norm(s):
    ty = s["x"].dtype
    h = (s["x"].float() + s["residual"].float()).to(ty)
    hf, w = h.float(), s["weight"]
    if s["case"]["mode"] == "int8":
        # 64 bits: which of two whole numbers a value rounds to must not hang on the order of a sum
        v = h.double() * w.double()
        most = v.abs().amax(1, keepdim=True)
        q = torch.where(most > 0, 127 * v / most, 0.0).round().to(torch.int8)
        rstd = (hf.square().mean(1, keepdim=True) + EPS).rsqrt()
        return [h, q, (most.float() * rstd / 127).squeeze(1)]
    rstd = (hf.square().mean(1, keepdim=True) + EPS).rsqrt()
    y = (hf * rstd * w).to(ty)
    dy = s["grad_out"].float()
    unit = hf * rstd
    dot = (dy * w * unit).mean(1, keepdim=True)
    gx = (rstd * (dy * w - unit * dot) + s["grad_summed"].float()).to(ty)
    return [h, y, gx, (dy * unit).sum(0)]


def plain_ffn(s):
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    g, u = x @ wg.t(), x @ wu.t()
    if s["x"].dtype == torch.int8:
        row = s["x_scale"][:, None]
        g, u = g * row * s["gate_scale"], u * row * s["up_scale"]
    sig = 1 / (1 + torch.exp(-g))
    act = g * sig
    if s["case"]["mode"] == "forward":
        return [(act * u).to(torch.bfloat16 if s["x"].dtype == torch.int8 else s["x"].dtype)]
    ty, dh = s["x"].dtype, s["grad_out"].float()
    dg = dh * u * sig * (1 + g * (1 - sig))
    du = dh * act
    return [(act * u).to(ty), (dg @ wg + du @ wu).to(ty), (dg.t() @ x).to(ty), (du.t() @ x).to(ty)]


def plain_ce(s):
    x, w, ty = s["x"].float(), s["weight"].float(), s["x"].dtype
    live = s["targets"] >= 0
    at = s["targets"].clamp_min(0)[:, None]
    z = x @ w.t()
    most = z.amax(1, keepdim=True)
    lse = most + torch.exp(z - most).sum(1, keepdim=True).log()
    loss = torch.where(live, (lse - z.gather(1, at)).squeeze(1), 0.0)
    if s["case"]["mode"] == "forward":
        return [loss, lse.squeeze(1)]
    p = torch.exp(z - lse)
    p.scatter_add_(1, at, torch.full_like(lse, -1.0))
    p *= torch.where(live, s["grad_loss"], 0.0)[:, None]
    return [loss, lse.squeeze(1), (p @ w).to(ty), (p.t() @ x).to(ty)]


def plain_clip(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    factor = (MAX_NORM / (norm + 1e-6)).clamp_max(1.0)
    return [norm.reshape(1)] + [(g.float() * factor).to(g.dtype) for g in s["grads"]]


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}[case["type"]]
    if case["op"] == "norm":
        r, c = case["rows"], case["cols"]
        if case["mode"] == "int8":  # x, residual, weight; h, q, scale
            return {"bytes": r * c * (3 * size + 1) + 4 * c + 4 * r, "flops": 0}
        # forward x, residual, weight; h, y.  Backward: grad_out, grad_summed, h, weight; grad_in, grad_weight
        return {"bytes": r * c * 8 * size + 12 * c, "flops": 0}
    if case["op"] == "ffn":
        t, d, f = case["tokens"], case["d"], case["f"]
        if case["mode"] == "forward":
            return {"bytes": size * (t * d + 2 * f * d) + 2 * t * f, "flops": 4 * t * d * f}
        # x, both weights, grad_out; out, grad_x and both weights' gradients
        return {"bytes": size * (2 * t * d + 4 * f * d + 2 * t * f), "flops": 12 * t * d * f}
    if case["op"] == "ce":
        t, d, v = case["tokens"], case["d"], case["vocab"]
        if case["mode"] == "forward":
            return {"bytes": size * (t * d + v * d) + 16 * t, "flops": 2 * t * d * v}
        # three products; the one that makes the logits again is not needed by the mathematics
        return {"bytes": 2 * size * (t * d + v * d) + 20 * t, "flops": 6 * t * d * v}
    # every gradient read once, every clipped one written once
    return {"bytes": 2 * size * sum(tensor_sizes(case)), "flops": 0}


def exact(case, seed):
    """The same outputs from the definitions, in 64 bits."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    d = {k: v.double() for k, v in s.items() if torch.is_tensor(v)}
    if case["op"] == "norm":
        # h is what the operator stores: the sum of two stored values, in their type
        h = (d["x"] + d["residual"]).to(s["x"].dtype).double()
        rms = (h.pow(2).sum(1) / case["cols"] + EPS).sqrt()[:, None]
        if case["mode"] == "int8":
            top = (h * d["weight"]).abs().max(1).values[:, None]
            step = torch.where(top > 0, top, 1.0)
            q = torch.round((h * d["weight"]) * 127 / step)
            return [h, q.to(torch.int8), (top / rms / 127)[:, 0]]
        a = d["grad_out"] * d["weight"]
        n = h / rms
        gx = d["grad_summed"] + (a - n * (a * n).sum(1)[:, None] / case["cols"]) / rms
        return [h, n * d["weight"], gx, (n * d["grad_out"]).sum(0)]
    if case["op"] == "ffn":
        g, u = torch.mm(d["x"], d["w_gate"].t()), torch.mm(d["x"], d["w_up"].t())
        if case["type"] == "i8":
            g *= d["x_scale"][:, None] * d["gate_scale"][None]
            u *= d["x_scale"][:, None] * d["up_scale"][None]
        s1 = torch.sigmoid(g)
        if case["mode"] == "forward":
            return [g * s1 * u]
        dg = d["grad_out"] * u * (s1 + g * s1 * (1 - s1))
        du = d["grad_out"] * g * s1
        gx = torch.mm(dg, d["w_gate"]) + torch.mm(du, d["w_up"])
        return [g * s1 * u, gx, torch.mm(dg.t().contiguous(), d["x"]), torch.mm(du.t().contiguous(), d["x"])]
    if case["op"] == "ce":
        z = torch.mm(d["x"], d["weight"].t())
        lse = torch.logsumexp(z, 1)
        rows = torch.nonzero(s["targets"] >= 0)[:, 0]
        loss = torch.zeros_like(lse)
        loss[rows] = lse[rows] - z[rows, s["targets"][rows]]
        if case["mode"] == "forward":
            return [loss, lse]
        z.sub_(lse[:, None]).exp_()
        z[rows, s["targets"][rows]] -= 1
        scale = torch.zeros_like(lse)
        scale[rows] = d["grad_loss"][rows]
        z.mul_(scale[:, None])
        return [loss, lse, torch.mm(z, d["weight"]), torch.mm(z.t(), d["x"])]
    total = sum(g.double().pow(2).sum() for g in s["grads"]).sqrt()
    factor = min(1.0, MAX_NORM / (float(total) + 1e-6))
    return [total.reshape(1)] + [g.double() * factor for g in s["grads"]]
