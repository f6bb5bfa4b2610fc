"""The language-model operators at the edges of their ranges, against their definitions in 64 bits:
values near the ends of a type, rows of zeros, dimensions past 32-bit offsets, calls without tokens.

Tolerances as in test_gpu_operators.py: U = 2^-24 for an fp32 operation, half(T) for a rounding to T,
tiny(T) for one among T's subnormal numbers."""
import numpy as np
import pytest

from hc_amd import runtime as rt

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_operators import TYPES, U, act_reference, dev, empty, f64, half, near, normal, strided, tiny  # noqa: E402


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
