"""The precision of a packed Linear layer's activations goes with the compressed state dict."""
import io

import pytest
import torch
from torch import nn


def packed(tmq, seed):
    torch.manual_seed(seed)
    lin = tmq.Linear(32, 20, ctrl=tmq.QuantizationControl(), quant_mode=tmq.QuantMode.TERNARY)
    lin.weight = nn.Parameter(torch.randint(0, 1 << 20, (32, 2), dtype=torch.int32), requires_grad=False)
    lin.original_shape = (20, 32)
    lin.tensor_type = tmq.TensorType.COMPACT_TERNARY_32BIT
    return nn.Sequential(nn.ReLU(), lin)


def through_a_file(state):
    buf = io.BytesIO()
    torch.save(state, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)


@pytest.mark.parametrize("bits", [None, 8])
def test_the_setting_is_saved_and_restored(bits):
    from tmq_b200 import tmq
    model = packed(tmq, 1)
    tmq.set_activation_bits(model, bits)
    state = through_a_file(tmq.compressed_state_dict(model))
    fresh = packed(tmq, 2)
    tmq.load_compressed_state_dict(fresh, state)
    assert fresh[1].activation_bits == bits and fresh[1].compact
    assert torch.equal(fresh[1].weight, model[1].weight)


def test_a_state_dict_without_the_setting_leaves_it():
    from tmq_b200 import tmq
    state = tmq.compressed_state_dict(packed(tmq, 1))
    assert "tmq.activation_bits" not in state._metadata["1"]
    fresh = packed(tmq, 2)
    tmq.set_activation_bits(fresh, 8)
    tmq.load_compressed_state_dict(fresh, state)
    assert fresh[1].activation_bits == 8
