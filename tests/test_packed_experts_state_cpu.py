"""What a stack of experts keeps: its weights, tables and precision in the state dict, its tables in fp32.  No GPU: the packed
words are stand-ins."""
import copy

import pytest
import torch
from torch import nn

N_IN, N_OUT = 40, 24


@pytest.fixture
def tmq(monkeypatch):
    from tmq_b200 import ops, tmq
    monkeypatch.setattr(tmq, "_require_cuda", lambda t, what: None)

    def words(packed, columns, fmt):
        row = packed[:, 0].repeat(8)[:ops.prepack_row_words(packed.shape[0], fmt)]
        return (row + 1000 * fmt).repeat(columns, 1)

    monkeypatch.setattr(ops, "prepack", words)
    return tmq


def layers(tmq, seed, bias=True, scale=1.0, count=3, n_in=N_IN):
    torch.manual_seed(seed)
    made = []
    for e in range(count):
        lin = tmq.Linear(n_in, N_OUT, bias=bias, ctrl=tmq.QuantizationControl(), quant_mode=tmq.QuantMode.TERNARY)
        if bias:
            lin.bias.data.normal_()
        lin.weight = nn.Parameter(torch.randint(0, 1 << 20, (n_in, 2), dtype=torch.int32), requires_grad=False)
        lin.original_shape = (N_OUT, n_in)
        lin.compact = True
        lin._scale_dirty = False
        lin.post_scale_imm = scale * (1 + e / 7)
        made.append(lin)
    return made


def same(a, b):
    for name in ("weights", "scales", "biases"):
        x, y = getattr(a, name), getattr(b, name)
        assert (x is None) == (y is None) and (x is None or torch.equal(x, y)), name
    assert a.activation_bits == b.activation_bits


@pytest.mark.parametrize("bits", [None, 8])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scale", [1.0, 0.3])
def test_the_state_dict_restores_everything(tmq, bits, bias, scale, tmp_path):
    lay = layers(tmq, 1, bias, scale)
    if scale == 1.0:
        for lin in lay:
            lin.post_scale_imm = 1.0
    model = nn.ModuleDict({"experts": tmq.PackedExperts(lay, activation_bits=bits)})
    torch.save(model.state_dict(), tmp_path / "m.pt")
    for other_bias, other_scale, other_bits in ((True, 0.7, 8), (False, 0.7, None)):
        fresh = nn.ModuleDict({"experts": tmq.PackedExperts(layers(tmq, 2, other_bias, other_scale), activation_bits=other_bits)})
        fresh.load_state_dict(torch.load(tmp_path / "m.pt", weights_only=True))
        same(fresh["experts"], model["experts"])


def test_other_experts_are_refused(tmq):
    state = tmq.PackedExperts(layers(tmq, 1)).state_dict()
    for lay in (layers(tmq, 2, count=2), layers(tmq, 2, n_in=N_IN + 1)):
        module = tmq.PackedExperts(lay)
        before = copy.deepcopy(module)
        with pytest.raises(RuntimeError):
            module.load_state_dict(state)
        same(module, before)
    module = tmq.PackedExperts(layers(tmq, 2))
    with pytest.raises(RuntimeError):
        module.load_state_dict({k: v for k, v in state.items() if k != "weights"})


def test_a_state_dict_from_before_leaves_the_stack(tmq):
    model = nn.Sequential(tmq.PackedExperts(layers(tmq, 1)), nn.Linear(3, 3))
    before = copy.deepcopy(model[0])
    old = model[1].state_dict(prefix="1.")
    old._metadata[""] = {"version": 1}
    old._metadata["0"] = {"version": 1}
    model.load_state_dict(old)
    same(model[0], before)


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.float16), lambda m: m.double()])
def test_casts_leave_the_tables_alone(tmq, cast):
    model = nn.Sequential(tmq.PackedExperts(layers(tmq, 3, scale=0.3)), nn.Linear(2, 2))
    before = copy.deepcopy(model[0])
    cast(model)
    assert model[0].scales.dtype == model[0].biases.dtype == torch.float32 and model[1].weight.dtype != torch.float32
    same(model[0], before)


def test_the_default_dtype_does_not_reach_the_tables(tmq):
    lay = layers(tmq, 4, scale=0.3)
    lay[0].bias = None
    want = tmq.PackedExperts(lay)
    torch.set_default_dtype(torch.bfloat16)
    try:
        got = tmq.PackedExperts(lay)
    finally:
        torch.set_default_dtype(torch.float32)
    same(got, want)
    assert got.scales.dtype == got.biases.dtype == torch.float32
