"""CPU checks of the weights that the expert-parallel layer takes: any object with the bf16 tensors, and
not the 8-bit ones."""
from types import SimpleNamespace

import pytest
import torch


@pytest.fixture
def ep(monkeypatch):
    from moe_b200 import ep
    monkeypatch.setattr(ep.dist, "get_world_size", lambda group=None: 1)
    monkeypatch.setattr(ep.dist, "get_rank", lambda group=None: 0)
    return ep


def test_any_object_with_the_tensors(ep):
    w1, w2 = torch.zeros(4, 64, 32, dtype=torch.bfloat16), torch.zeros(4, 32, 32, dtype=torch.bfloat16)
    w = SimpleNamespace(w1=w1, w2=w2, num_experts=4, hidden=32, ffn=32)
    layer = ep.MoELayerEP(w, num_experts=4, topk=2)
    assert layer.w is w and layer.plan.num_groups == 4


def test_8_bit_weights_are_refused(ep):
    import moe_b200
    q = moe_b200.Fp8Tensor(torch.zeros(4, 256, 32), torch.zeros(4, 2, 1))
    with pytest.raises(ValueError, match="bf16 rows"):
        ep.MoELayerEP(moe_b200.MoEWeightsFp8(q, q), num_experts=4)
