"""What the 8-bit operators refuse of tensors on the GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from tf_depth_estimation_amd import int8

pytestmark = pytest.mark.gpu


def calls():
    conv = int8.Conv8(torch.ones(1, 1, 8, 4, device="cuda"))
    beta = torch.zeros(8, device="cuda")
    _, tape = int8.bn_relu_forward(torch.randn(16, 8, device="cuda"), beta)
    return {"quantize": int8.quantize_rows, "conv": conv, "weights": lambda t: int8.Conv8(t.view(1, 1, 16, 8)),
            "forward": lambda t: int8.bn_relu_forward(t, beta),
            "beta": lambda t: int8.bn_relu_forward(torch.ones(16, 8, device="cuda"), t[0]),
            "backward": lambda t: int8.bn_relu_backward(tape, beta, t), "restore": lambda t: tape.restore(out=t)}


def test_forward_mode_tangents():
    """A dual tensor's tangent would be lost without a word."""
    x = torch.randn(16, 8, device="cuda")
    for name, f in calls().items():
        with forward_ad.dual_level():
            f(x)                                              # (a level alone changes nothing)
            with pytest.raises(ValueError, match="tangent"):
                f(forward_ad.make_dual(x.clone(), torch.ones_like(x)))
        with pytest.raises(ValueError, match="gradient"):
            f(x.clone().requires_grad_())
        with torch.no_grad():
            f(x.clone().requires_grad_())
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(calls()["conv"], (x,), (torch.ones_like(x),))
