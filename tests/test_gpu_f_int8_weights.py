"""The 8-bit weight that is kept with a layer: what makes it stale, and what does not."""

import copy
import io

import pytest
import torch

from peco_b200.int8 import int8_weight, linear_int8, quantize_layer, quantize_rows

pytestmark = pytest.mark.gpu


def layer_in_8_bits():
    torch.manual_seed(0)
    layer = torch.nn.Linear(72, 40, device="cuda", dtype=torch.bfloat16)
    assert quantize_layer(layer)
    assert int8_weight(layer) is not None
    return layer


def repoint(layer):
    layer.weight.data = layer.weight.data * 2


def repoint_within(layer):
    layer.weight.data = layer.weight.data.new_zeros(2, 40, 72)[0]
    quantize_layer(layer)
    layer.weight.data = layer.weight.data.as_strided((40, 72), (72, 1), 40 * 72)


def merge(layer):
    with torch.no_grad():
        layer.weight += 1


def replace(layer):
    layer.weight = torch.nn.Parameter(layer.weight.detach() * 2)


def there_and_back(layer):
    layer.cpu()
    layer.weight.data.mul_(2)
    layer.cuda()


@pytest.mark.parametrize("change", [repoint, repoint_within, merge, replace, there_and_back, lambda layer: layer.half(), lambda layer: layer.cpu()])
def test_a_changed_or_moved_weight_is_noticed(change):
    layer = layer_in_8_bits()
    change(layer)
    with pytest.raises(RuntimeError, match="quantise it again"):
        int8_weight(layer)
    if layer.weight.is_cuda:
        assert quantize_layer(layer)
        assert torch.equal(int8_weight(layer).values, quantize_rows(layer.weight.detach()).values)


def test_a_copied_layer_keeps_its_8_bit_weight():
    layer = layer_in_8_bits()
    with torch.no_grad():
        layer.weight.mul_(2)  # a version that a copy's weight does not have
    quantize_layer(layer)
    twin = copy.deepcopy(layer)
    x = torch.randn(5, 72, device="cuda").bfloat16()
    with torch.no_grad():
        out = linear_int8(x, int8_weight(layer), layer.bias)
        layer.weight.zero_()
        assert torch.equal(linear_int8(x, int8_weight(twin), twin.bias), out)
        twin.weight.mul_(2)
    stored = io.BytesIO()
    torch.save(copy.deepcopy(twin), stored)
    for stale in (layer, twin, copy.deepcopy(twin), torch.load(io.BytesIO(stored.getvalue()), weights_only=False)):
        with pytest.raises(RuntimeError, match="quantise it again"):
            int8_weight(stale)


def test_a_stored_layer_keeps_its_8_bit_weight():
    layer, x = layer_in_8_bits(), torch.randn(5, 72, device="cuda").bfloat16()
    stored = io.BytesIO()
    torch.save(layer, stored)
    again = torch.load(io.BytesIO(stored.getvalue()), weights_only=False)
    with torch.no_grad():
        assert torch.equal(linear_int8(x, int8_weight(again)), linear_int8(x, int8_weight(layer)))


def test_weights_made_for_inference_alone():
    """Tensors of inference mode have no version."""
    with torch.inference_mode():
        layer = layer_in_8_bits()
        x = torch.randn(5, 72, device="cuda").bfloat16()
        assert torch.equal(linear_int8(x, int8_weight(layer)), linear_int8(x, quantize_rows(layer.weight)))
        repoint(layer)
        with pytest.raises(RuntimeError, match="quantise it again"):
            int8_weight(layer)
