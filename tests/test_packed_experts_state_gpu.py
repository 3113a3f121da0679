"""Experts written and read back answer with the same bits, on a cast module too."""
import pytest
import torch
from torch import nn

from test_activation_bits_gpu import packed_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [None, 8])
def test_saved_experts_answer_the_same(bits, tmp_path):
    import tmq_b200 as tmq
    made = lambda seed, **kw: [packed_linear(tmq, 200, 96, seed + e, **kw)[0] for e in range(3)]
    model = nn.Sequential(tmq.PackedExperts(made(1, post_scale=True), activation_bits=bits))
    x = torch.randn(40, 200, device="cuda").to(torch.bfloat16)
    off = torch.tensor([0, 11, 11, 40], device="cuda")
    y = model[0](x, off)
    torch.save(model.state_dict(), tmp_path / "m.pt")
    fresh = nn.Sequential(tmq.PackedExperts(made(9, bias=False), activation_bits=None if bits else 8))
    assert not torch.equal(fresh[0](x, off), y)
    fresh.load_state_dict(torch.load(tmp_path / "m.pt", weights_only=True))
    assert torch.equal(fresh[0](x, off), y)
    assert torch.equal(fresh.half()[0](x, off), y)
