"""rms_norm and the codes behind it at the ends of what they take, and what its results' gradients are."""
import pytest
import torch

import int8_reference as ref
from test_gpu_int8 import F32, randn

pytestmark = pytest.mark.gpu


# ---- what the sum's gradient is --------------------------------------------------------------------------------------------------

def test_the_sum_wants_no_gradient_of_a_weight():
    """x + residual does not depend on the weight: with the weight the only leaf the sum is a constant, and the next block's norm takes it in
    8 bits; with x or the residual a leaf it is none."""
    import mflux_amd
    from mflux_amd import nn

    norm = nn.RMSNorm(64, 1e-6, device="cuda", dtype=F32)
    x, h, dy = randn(1, 5, 64), randn(2, 5, 64), randn(3, 5, 64)
    y, s = norm(x, residual=h)
    assert y.requires_grad and not s.requires_grad and s.grad_fn is None
    want = ref.rms_norm(ref.total(x, h), norm.weight, 1e-6, dy)
    ref.check("dw", torch.autograd.grad(y, norm.weight, dy)[0], *want["dw"])
    q, sc, total = norm.int8(x, residual=s)
    assert torch.equal(total, s + x) and not total.requires_grad
    for leaf in ("x", "h"):
        x1, h1 = (t.clone().requires_grad_(n == leaf) for n, t in (("x", x), ("h", h)))
        y, s = mflux_amd.rms_norm(x1, norm.weight, residual=h1)
        assert y.requires_grad and s.requires_grad
        d, = torch.autograd.grad(s, x1 if leaf == "x" else h1, dy)
        assert torch.equal(d, dy)
