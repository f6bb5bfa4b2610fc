"""What the language-model operators refuse, without a GPU: the plans' checks on host
arrays, and the entry points' own checks on a queue that has nothing but an error
callback (every call here is refused before anything is launched)."""
import ctypes as C

import numpy as np
import pytest

from hc_amd import runtime as rt


class HostOnly:
    queue = None


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(rt, "default_context", lambda *a: HostOnly)
    monkeypatch.setattr(rt, "_workspace", lambda nbytes, ctx: None)


def f32(*shape):
    return np.zeros(shape, np.float32)


def f16(*shape):
    return np.zeros(shape, np.float16)


def i8(*shape):
    return np.zeros(shape, np.int8)


PLANS = [
    ("x: element type", lambda: rt.plan_add_rms_norm(i8(2, 8), None, None, i8(2, 8))),
    ("residual: shape", lambda: rt.plan_add_rms_norm(f16(2, 8), f16(2, 9), None, f16(2, 8))),
    ("residual: element type", lambda: rt.plan_add_rms_norm(f16(2, 8), f32(2, 8), None, f16(2, 8))),
    ("out: element type", lambda: rt.plan_add_rms_norm(f16(2, 8), None, None, f32(2, 8))),
    ("out: shape", lambda: rt.plan_add_rms_norm(f16(2, 8), None, None, f16(3, 8))),
    ("weight: 8 contiguous", lambda: rt.plan_add_rms_norm(f16(2, 8), None, f32(7), f16(2, 8))),
    ("weight: element type", lambda: rt.plan_add_rms_norm(f32(2, 8), None, f16(8), f32(2, 8))),
    ("rows must be contiguous", lambda: rt.plan_add_rms_norm(f16(2, 16)[:, ::2], None, None, f16(2, 8))),
    ("negative stride", lambda: rt.plan_add_rms_norm(f16(2, 8)[::-1], None, None, f16(2, 8))),
    ("scale: 2 contiguous", lambda: rt.plan_add_rms_norm(f16(2, 8), None, None, i8(2, 8), scale=f32(3))),
    ("summed: element type", lambda: rt.plan_add_rms_norm_backward(f16(2, 8), f32(2, 8), None, f32(2), f16(2, 8))),
    ("rstd: 2 contiguous", lambda: rt.plan_add_rms_norm_backward(f16(2, 8), f16(2, 8), None, f32(1), f16(2, 8))),
    ("grad_weight: the weight's", lambda: rt.plan_add_rms_norm_backward(
        f16(2, 8), f16(2, 8), f32(8), f32(2), f16(2, 8), f16(8))),
    ("x: element type", lambda: rt.plan_gated_ffn(f32(2, 8), f32(4, 8), f32(4, 8), f32(2, 4))),
    ("w_gate: rows of 9", lambda: rt.plan_gated_ffn(f16(2, 8), f16(4, 9), f16(4, 9), f16(2, 4))),
    ("w_up: shape", lambda: rt.plan_gated_ffn(f16(2, 8), f16(4, 8), f16(5, 8), f16(2, 4))),
    ("out: shape", lambda: rt.plan_gated_ffn(f16(2, 8), f16(4, 8), f16(4, 8), f16(2, 5))),
    ("activation 'relu'", lambda: rt.plan_gated_ffn(f16(2, 8), f16(4, 8), f16(4, 8), f16(2, 4), activation="relu")),
    ("three scales", lambda: rt.plan_gated_ffn(i8(2, 8), i8(4, 8), i8(4, 8), f16(2, 4))),
    ("three scales", lambda: rt.plan_gated_ffn(f16(2, 8), f16(4, 8), f16(4, 8), f16(2, 4), scales=(f32(2), f32(4), f32(4)))),
    ("up_scale: 4 contiguous", lambda: rt.plan_gated_ffn(i8(2, 8), i8(4, 8), i8(4, 8), f16(2, 4),
                                                         scales=(f32(2), f32(4), f32(5)))),
    ("out: element type", lambda: rt.plan_gated_ffn(i8(2, 8), i8(4, 8), i8(4, 8), i8(2, 4), scales=(f32(2), f32(4), f32(4)))),
    ("x: 3 rows", lambda: rt.plan_gated_ffn_backward(f16(2, 4), f16(3, 8), f16(4, 8), f16(4, 8), f16(2, 4), f16(2, 4))),
    ("gate: shape", lambda: rt.plan_gated_ffn_backward(f16(2, 4), f16(2, 8), f16(4, 8), f16(4, 8), f16(2, 5), f16(2, 4))),
    ("grad_w_up: shape", lambda: rt.plan_gated_ffn_backward(
        f16(2, 4), f16(2, 8), f16(4, 8), f16(4, 8), f16(2, 4), f16(2, 4), grad_w_up=f16(8, 4))),
    ("weight: rows of 9", lambda: rt.plan_linear_cross_entropy(f16(2, 8), f16(5, 9), np.zeros(2, np.int64), f32(2), f32(2))),
    ("targets: element type", lambda: rt.plan_linear_cross_entropy(f16(2, 8), f16(5, 8), f32(2), f32(2), f32(2))),
    ("targets: 2 contiguous", lambda: rt.plan_linear_cross_entropy(
        f16(2, 8), f16(5, 8), np.zeros(4, np.int64)[::2], f32(2), f32(2))),
    ("lse: element type", lambda: rt.plan_linear_cross_entropy(f16(2, 8), f16(5, 8), np.zeros(2, np.int32), f32(2), f16(2))),
    ("negative piece", lambda: rt.plan_linear_cross_entropy_backward(
        f16(2, 8), f16(5, 8), np.zeros(2, np.int32), f32(2), f32(2), f16(2, 8), f16(5, 8), piece=-1)),
    ("grad_weight: shape", lambda: rt.plan_linear_cross_entropy_backward(
        f16(2, 8), f16(5, 8), np.zeros(2, np.int32), f32(2), f32(2), f16(2, 8), f16(8, 5))),
    ("one output per gradient", lambda: rt.plan_clip_grad_norm([f32(3)], [], f32(1), 1.0)),
    ("tensor 0", lambda: rt.plan_clip_grad_norm([f32(3)], [f16(3)], f32(1), 1.0)),
    ("tensor 1 must be contiguous", lambda: rt.plan_clip_grad_norm([f32(3), f32(4, 4)[:, :2]], [f32(3), f32(4, 2)], f32(1), 1.0)),
    ("tensor 0", lambda: rt.plan_clip_grad_norm([i8(3)], [i8(3)], f32(1), 1.0)),
]


@pytest.mark.parametrize("k", range(len(PLANS)))
def test_plans_refuse(host, k):
    match, call = PLANS[k]
    with pytest.raises(rt.HcRuntimeError, match=match):
        call()


# ---- the C entry points -------------------------------------------------------
class FakeQueue:
    """The memory of a queue whose device has an error callback and nothing else
    (Queue begins with its device, Device with the callback and its context)."""

    def __init__(self):
        self.messages = []
        self.cb = rt.ERROR_CALLBACK(lambda ctx, sev, text: self.messages.append(text.decode()))
        self.device = (C.c_uint64 * 128)()
        self.device[0] = C.cast(self.cb, C.c_void_p).value
        self.memory = (C.c_uint64 * 2)(C.addressof(self.device), 0)
        self.ptr = C.addressof(self.memory)


P = 1 << 20             # an address that is never touched
F32, F16, BF16, I8, I32, I64 = rt.F32, rt.F16, rt.BF16, rt.I8, rt.I32, rt.I64


def norm(q, ty=F16, x=P, ldx=8, r=None, w=None, wt=F32, eps=1e-6, summed=None, out=P, ot=F16, ldo=8, scale=None,
         rstd=None, rows=2, cols=8):
    return rt.hcamdLaunchAddRmsNorm(q, ty, x, ldx, r, 8, w, wt, eps, summed, 8, out, ot, ldo, scale, rstd, rows, cols)


def norm_back(q, ty=F16, g=P, gw=None, wt=F32, rows=2, cols=8, work=None, have=0, rstd=P):
    return rt.hcamdLaunchAddRmsNormBackward(q, ty, g, 8, P, 8, None, wt, rstd, None, 8, P, 8, gw, rows, cols, work, have)


def ffn(q, ty=F16, x=P, ldx=8, xs=None, act=0, ot=F16, gate=None, t=2, d=8, f=4, out=P, wu=P, work=None, have=0):
    return rt.hcamdLaunchGatedFfn(q, ty, x, ldx, xs, P, 1 << 18, xs, wu, 1 << 18, xs, act, out, ot, 4, gate, 4, None, 4, t, d, f, work, have)


def ffn_back(q, ty=F16, g=P, x=P, w=P, gx=P, work=None, have=0, t=2, d=8, f=4, act=0):
    return rt.hcamdLaunchGatedFfnBackward(q, ty, g, 4, x, 8, w, 8, w, 8, P, 4, P, 4, act, gx, 8, None, 8, P, 8, t, d, f, work, have)


def ce(q, ty=F16, x=P, tt=I64, targets=P, work=None, have=0, t=2, d=8, v=5, loss=P):
    return rt.hcamdLaunchLinearCrossEntropy(q, ty, x, 8, P, 8, targets, tt, loss, P, t, d, v, work, have)


def ce_back(q, ty=F16, gx=P, work=None, have=0, t=2, piece=0, gl=P):
    return rt.hcamdLaunchLinearCrossEntropyBackward(q, ty, P, 8, P, 8, P, I32, P, gl, gx, 8, P, 8, t, 8, 5, piece, work, have)


def clip(q, table=None, n=1, most=1.0, norm_=P, work=P, have=1 << 20):
    table = table or [(P, P, 4, F32)]
    return rt.hcamdLaunchClipGradNorm(q, (rt.ClipTensor * len(table))(*table), n, most, norm_, work, have)


ENTRIES = [
    ("element type 6", norm, dict(ty=I8)), ("output type 0", norm, dict(ot=F32)), ("weight type 2", norm, dict(w=P, wt=BF16)),
    ("eps must not", norm, dict(eps=-1.0)), ("eps must not", norm, dict(eps=float("nan"))), ("x is null", norm, dict(x=None)),
    ("x is not aligned", norm, dict(x=P + 1)), ("x: leading dimension smaller", norm, dict(ldx=7)),
    ("x: leading dimension out of range", norm, dict(ldx=1 << 50)), ("out is null", norm, dict(out=None)),
    ("scale is null", norm, dict(ot=I8)), ("a scale needs", norm, dict(scale=P)), ("rstd is not aligned", norm, dict(rstd=P + 2)),
    ("rows without elements", norm, dict(cols=0)), ("a dimension exceeds", norm, dict(rows=1 << 31)),
    ("summed is not aligned", norm, dict(summed=P + 1)),
    ("element type 6", norm_back, dict(ty=I8)), ("weight type 2", norm_back, dict(wt=BF16)),
    ("grad_out is null", norm_back, dict(g=None)), ("workspace of 0 bytes, 64 needed", norm_back, dict(gw=P)),
    ("aligned to 256", norm_back, dict(gw=P, work=P + 16, have=1024)), ("rstd is null", norm_back, dict(rstd=None)),
    ("element type 0", ffn, dict(ty=F32)), ("output type 2", ffn, dict(ot=BF16)), ("activation 2", ffn, dict(act=2)),
    ("inner dimension must", ffn, dict(d=0)), ("x_scale is null", ffn, dict(ty=I8)), ("scales belong", ffn, dict(xs=P)),
    ("pre-activations", ffn, dict(ty=I8, xs=P, gate=P)), ("131072", ffn, dict(ty=I8, xs=P, d=131073, ldx=1 << 18)),
    ("output type 6", ffn, dict(ty=I8, xs=P, ot=I8)), ("out is null", ffn, dict(out=None)), ("w_up is null", ffn, dict(wu=None)),
    ("element type 6", ffn_back, dict(ty=I8)), ("grad_out is null", ffn_back, dict(g=None)), ("x is null", ffn_back, dict(x=None)),
    ("w_gate is null", ffn_back, dict(w=None)), ("empty dimension", ffn_back, dict(f=0)), ("workspace of 0 bytes", ffn_back, {}),
    ("workspace of 0 bytes", ffn, dict(t=800, d=7)), ("aligned to 256", ffn, dict(t=800, d=7, work=P + 16, have=1 << 20)),
    ("workspace of 0 bytes", ffn, dict(ty=I8, xs=P, t=800, ldx=16, d=9)), ("activation -1", ffn_back, dict(act=-1)),
    ("element type 0", ce, dict(ty=F32)), ("target type 0", ce, dict(tt=F32)), ("targets is null", ce, dict(targets=None)),
    ("targets is not aligned", ce, dict(targets=P + 4)), ("empty dimension", ce, dict(v=0)), ("workspace of 0 bytes", ce, {}),
    ("loss is null", ce, dict(loss=None)),
    ("element type 6", ce_back, dict(ty=I8)), ("grad_loss is null", ce_back, dict(gl=None)), ("a piece of", ce_back, dict(piece=1 << 32)),
    ("workspace of 0 bytes", ce_back, {}), ("grad_x is not aligned", ce_back, dict(gx=P + 1)),
    ("must not be negative", clip, dict(most=-1.0)), ("must not be negative", clip, dict(most=float("nan"))),
    ("norm is null", clip, dict(norm_=None)), ("workspace of 0 bytes", clip, dict(work=None)),
    ("type 6", clip, dict(table=[(P, P, 4, I8)])), ("a tensor is null", clip, dict(table=[(None, P, 4, F32)])),
    ("clipped tensor is not aligned", clip, dict(table=[(P, P + 1, 4, F16)])),
    ("too many elements", clip, dict(table=[(P, P, 1 << 41, F16)])),
]


@pytest.mark.parametrize("k", range(len(ENTRIES)))
def test_entry_points_refuse(k):
    match, call, kw = ENTRIES[k]
    q = FakeQueue()
    assert call(q.ptr, **kw) == 1
    assert len(q.messages) == 1 and match in q.messages[0], q.messages


Q = [P + (k << 24) for k in range(1, 9)]    # addresses apart from P and from each other
ALIASES = [
    ("two outputs", lambda q: norm(q, out=P, summed=P)),
    ("two outputs", lambda q: norm(q, ot=I8, out=Q[0], scale=Q[1], rstd=Q[1])),
    ("an output is an input", lambda q: norm(q, x=P, ot=I8, out=P, scale=Q[1])),
    ("an output is an input", lambda q: norm(q, x=Q[0], w=Q[1], out=Q[1])),
    ("in place with another", lambda q: norm(q, x=P, out=P, ldo=16)),
    ("in place with another", lambda q: norm(q, x=P, ldx=16, out=Q[0], summed=P)),
    ("an output is an input", lambda q: norm_back(q, gw=None)),              # grad_in is summed
    ("two outputs", lambda q: rt.hcamdLaunchGatedFfn(q, F16, P, 8, None, Q[0], 8, None, Q[1], 8, None, 0, Q[2], F16, 4,
                                                     Q[3], 4, Q[3], 4, 2, 8, 4, None, 0)),
    ("an output is an input", lambda q: rt.hcamdLaunchGatedFfn(q, F16, P, 8, None, Q[0], 8, None, Q[1], 8, None, 0, P, F16, 8,
                                                               None, 8, None, 8, 2, 8, 8, None, 0)),
    ("an output is an input", lambda q: rt.hcamdLaunchGatedFfnBackward(q, F16, Q[0], 4, P, 8, Q[1], 8, Q[2], 8, Q[3], 4, Q[4], 4,
                                                                       0, P, 8, None, 8, Q[5], 8, 2, 8, 4, Q[6], 1 << 20)),
    ("two outputs", lambda q: rt.hcamdLaunchGatedFfnBackward(q, F16, Q[0], 4, P, 8, Q[1], 8, Q[2], 8, Q[3], 4, Q[4], 4, 0, None,
                                                             8, Q[5], 8, Q[5], 8, 2, 8, 4, Q[6], 1 << 20)),
    ("two outputs", lambda q: rt.hcamdLaunchLinearCrossEntropy(q, F16, Q[0], 8, Q[1], 8, Q[2], I64, P, P, 2, 8, 5, Q[3], 1 << 20)),
    ("an output is an input", lambda q: rt.hcamdLaunchLinearCrossEntropyBackward(
        q, F16, Q[0], 8, Q[1], 8, Q[2], I64, Q[3], Q[4], None, 8, Q[1], 8, 2, 8, 5, 0, Q[5], 1 << 20)),
]


@pytest.mark.parametrize("k", range(len(ALIASES)))
def test_shared_buffers_are_refused(k):
    match, call = ALIASES[k]
    q = FakeQueue()
    assert call(q.ptr) == 1
    assert len(q.messages) == 1 and match in q.messages[0], q.messages


def test_int8_sums_stay_below_their_limit():
    """131071 products of (-128)^2 fit 32 bits, one more does not."""
    q = FakeQueue()
    assert 131071 * 128 * 128 < 2 ** 31 <= 131072 * 128 * 128
    assert ffn(q.ptr, ty=I8, xs=P, d=131072, ldx=1 << 18) == 1 and "below 131072" in q.messages[0]


def test_nothing_to_do_is_no_error():
    q = FakeQueue()
    assert norm(q.ptr, rows=0, x=None, out=None) == 0
    assert ffn(q.ptr, t=0, x=None, out=None) == 0 and ffn(q.ptr, f=0) == 0
    assert ce(q.ptr, t=0, x=None) == 0
    assert not q.messages


def test_null_queue():
    for call in (norm, norm_back, ffn, ffn_back, ce, ce_back, clip):
        assert call(None) == 1


def test_workspace_sizes():
    """Sizes depend on the shape alone, hold what a call writes, and are 0 for empty or impossible shapes."""
    assert rt.hcamdAddRmsNormBackwardWorkspace(0, 8) == 0 and rt.hcamdGatedFfnBackwardWorkspace(0, 8, 8) == 0
    assert rt.hcamdGatedFfnBackwardWorkspace(1 << 40, 8, 8) == 0
    assert rt.hcamdLinearCrossEntropyBackwardWorkspace(0, 8, 8, 0) == 0
    for t, d, f in [(1, 1, 1), (7, 130, 3), (1000, 64, 257), (4096, 4096, 11264)]:
        assert rt.hcamdGatedFfnBackwardWorkspace(t, d, f) >= 4 * t * f
        for piece in (0, 1, 100):
            rows = min(f, max(piece, 8) if piece else f)
            assert rt.hcamdLinearCrossEntropyBackwardWorkspace(t, d, f, piece) >= 4 * t * d + (2 * t * rows if piece else 0)
