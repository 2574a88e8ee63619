"""Int8Linear on the device: adapters baked into its codes."""
import pytest
import torch

import int8_reference as ref
from test_gpu_int8 import BF16, F32, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K,N", [(64, 40), (77, 24)])
def test_adapters_are_baked_into_codes(K, N):
    """requantize=True: the codes and scales of the dequantised weight with the deltas, all adapters at once; what shares the layer's tensors
    follows."""
    import mflux_amd
    from mflux_amd import nn
    from mflux_amd.lora import FusedLoRALinear, LoRALinear, bake_and_strip_lora

    linear = nn.Linear(K, N, bias=True, device="cuda", dtype=BF16)
    with torch.no_grad():
        linear.weight.copy_(randn(1, N, K) * 0.05)
    base = linear.to_int8()
    loras = [LoRALinear.from_linear(linear, r=r, scale=s) for r, s in ((4, 0.5), (2, -2.0))]
    with torch.no_grad():
        for i, lora in enumerate(loras):
            lora.lora_A.copy_(randn(2 + i, *lora.lora_A.shape))
            lora.lora_B.copy_(randn(4 + i, *lora.lora_B.shape) * 0.01)
    full = mflux_amd.int8_dequantize(base.weight, base.scales, F32)
    deltas = sum(float(l.scale) * torch.matmul(l.lora_A.detach().float(), l.lora_B.detach().float()).t() for l in loras)
    q, s = mflux_amd.int8_quantize(full + deltas)
    weight, scales, x = base.weight, base.scales, randn(9, 5, K, dtype=BF16)
    with torch.no_grad():
        wrapped = FusedLoRALinear(base, loras)
        before = wrapped(x)
        out = bake_and_strip_lora(wrapped, requantize=True)
        assert out is base and base.weight is weight and base.scales is scales
        assert torch.equal(weight, q) and torch.equal(scales, s)
        after = base(x)
    # the wrapped layer's own error is x's rounding to codes; the baked one's weight is rounded once more: half a step of at most
    # max|row| / 127 in each of K values, and both results to bfloat16 (the wrapped one its two products and three sums as well)
    step = (full + deltas).abs().amax(1) / 127
    bound = x.double().abs().sum(1, keepdim=True) * step.double() / 2
    terms = x.double().abs() @ (full.abs() + sum(abs(l.scale) * l.lora_A.detach().abs().float() @ l.lora_B.detach().abs().float() for l in loras).t()).double().t()
    bound = bound + x.double().abs().amax(1, keepdim=True) / 254 * (deltas.abs().sum(1).double() + step.double() * K) + terms * 8 * ref.HALF[BF16] + 8 * ref.HALF[BF16] * linear.bias.detach().double().abs()
    assert bool(((after.double() - before.double()).abs() <= bound).all())


@pytest.mark.parametrize("how", ["move", "load", "assign", "copy"])
def test_a_moved_layer_multiplies_its_weight_where_it_is(how):
    """An input length that is no multiple of 16: a call allocates its x, its result and scratch, no second weight."""
    import copy

    from mflux_amd import nn

    K, N = 1001, 20000
    torch.manual_seed(1)
    layer = nn.Linear(K, N, bias=False, device="cuda", dtype=BF16).to_int8()
    x = randn(1, 2, K, dtype=BF16)
    want = layer(x)
    other = nn.Int8Linear(K, N, bias=False)
    state = {k: v.contiguous() for k, v in layer.state_dict().items()}
    if how == "move":
        other = layer.cpu().cuda()
    elif how == "copy":
        other = copy.deepcopy(layer)
    else:
        other.load_state_dict(state, assign=how == "assign")
        other = other.cuda()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = other(x)
    assert torch.cuda.max_memory_allocated() - before < N * K // 8
    assert torch.equal(y, want)
