"""What Int8Linear goes through on the host: adapters on it that are baked, moves, copies and loads.  No GPU."""
import pytest
import torch

from mflux_amd import nn
from mflux_amd.lora import FusedLoRALinear, LoRALinear, bake_and_strip_lora


def layer(K=32, N=8, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = nn.Int8Linear(K, N, bias=False)
    out.weight.copy_(torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8))
    out.scales.copy_(torch.rand(N, generator=g) * 1e-3)
    return out


def adapter(linear, delta=4.0):
    """An adapter whose product is `delta` everywhere, on a float layer of the same size."""
    lora = LoRALinear.from_linear(torch.nn.Linear(linear.input_dims, linear.output_dims, dtype=torch.float32), r=2, scale=1.0)
    with torch.no_grad():
        lora.lora_A.fill_(1.0)
        lora.lora_B.fill_(delta / 2)
    return lora


class Block(torch.nn.Module):
    def __init__(self, wrapper):
        super().__init__()
        self.first = LoRALinear.from_linear(torch.nn.Linear(32, 8, dtype=torch.float32), r=2)
        self.inner = torch.nn.ModuleList([wrapper])


@pytest.mark.parametrize("how", ["fused", "wrapped"])
def test_an_adapter_is_not_baked_into_codes(how):
    """A delta in units of the weight, added to codes, is neither scaled nor kept from wrapping round.  Refused, and before any other
    wrapper of the tree has been baked."""
    base = layer()
    if how == "fused":
        wrapper = FusedLoRALinear(base, [adapter(base)])
    else:
        wrapper = adapter(base)
        wrapper.linear = base
    for tree in (wrapper, Block(wrapper)):
        before = {k: v.clone() for k, v in tree.state_dict().items()}
        with pytest.raises(ValueError, match="requantize"):
            bake_and_strip_lora(tree)
        after = tree.state_dict()
        assert list(after) == list(before) and all(torch.equal(after[k], before[k]) for k in before)


def test_an_int8_layer_without_adapters_is_stripped():
    base = layer()
    before = base.weight.clone()
    assert bake_and_strip_lora(FusedLoRALinear(base, [])) is base
    # an adapter that carries an Int8Linear of its own is baked into the fused layer's base, which is what counts
    carrier = adapter(base, 0.5)
    carrier.linear = base
    lin = torch.nn.Linear(32, 8, dtype=torch.float32)
    weight = lin.weight.detach().clone()
    assert bake_and_strip_lora(FusedLoRALinear(lin, [carrier])) is lin
    assert torch.equal(lin.weight, weight + 0.5) and torch.equal(base.weight, before)


def padded(weight):
    """Rows of whole 16 bytes, to the last one's end."""
    N, K = weight.shape
    length = -(-K // 16) * 16
    return weight.stride(1) == 1 and weight.stride(0) % 16 == 0 and \
        weight.storage_offset() + (N - 1) * weight.stride(0) + length <= weight.untyped_storage().nbytes()


@pytest.mark.parametrize("K,N", [(77, 5), (1, 3), (100, 1), (64, 6)])
def test_a_weight_keeps_rows_of_whole_16_bytes(K, N):
    """However the layer came about: int8_matmul copies a weight that lies otherwise in every call."""
    import copy
    import io

    base = layer(K, N)
    assert padded(base.weight) and base.weight.shape == (N, K) and not base.weight.requires_grad
    codes = base.weight.clone().contiguous()
    state = {k: v.contiguous() for k, v in base.state_dict().items()}
    loaded, assigned = nn.Int8Linear(K, N, bias=False), nn.Int8Linear(K, N, bias=False)
    loaded.load_state_dict(state)
    assigned.load_state_dict(state, assign=True)
    file = io.BytesIO()
    torch.save(base, file)
    file.seek(0)
    meta = nn.Int8Linear(K, N, bias=False, device="meta").to_empty(device="cpu")
    meta.load_state_dict(state)
    for other in (loaded, assigned, copy.deepcopy(base), torch.load(file, weights_only=False), base.half(), base.to(torch.float32), meta,
                  copy.deepcopy(loaded).to(torch.bfloat16)):
        assert padded(other.weight) and other.weight.dtype == torch.int8 and torch.equal(other.weight, codes)
        assert torch.equal(other.scales, state["scales"])
    from mflux_amd.weights import update_module

    fresh = nn.Int8Linear(K, N, bias=False)
    update_module(fresh, state)
    assert padded(fresh.weight) and torch.equal(fresh.weight, codes)


def test_a_model_with_adapters_on_codes_is_not_saved_in_part(tmp_path):
    """The refusal comes before the first component is baked or written."""
    from mflux_amd import weights as W

    class Definition:
        @staticmethod
        def get_components():
            return [W.ComponentDefinition("first", "first"), W.ComponentDefinition("second", "second")]

    class Model:
        pass

    model, base = Model(), layer()
    model.first, model.second = Block(torch.nn.Identity()), Block(FusedLoRALinear(base, [adapter(base)]))
    before = model.first.first.linear.weight.detach().clone()
    with pytest.raises(ValueError, match="second.inner.0"):
        W.save_model(model, None, tmp_path, Definition)
    assert isinstance(model.first.first, LoRALinear) and torch.equal(model.first.first.linear.weight, before) and not list(tmp_path.iterdir())
