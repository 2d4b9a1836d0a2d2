"""A group table on a device given in any form that torch takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("device", ["cuda", "cuda:0", 0, torch.device("cuda"), torch.device("cuda", 0)])
def test_plan_device_forms(cuda_dev, device):
    import moe_b200
    x = torch.randn(40, 64, device=cuda_dev).to(torch.bfloat16)
    w = torch.randn(2, 32, 64, device=cuda_dev).to(torch.bfloat16)
    plan = moe_b200.GroupedGemmPlan(2, device).from_splits(torch.tensor([30, 10]))
    assert torch.equal(moe_b200.grouped_gemm(x, w, plan=plan), moe_b200.grouped_gemm(x, w, [30, 10]))
    assert plan.device_error() == 0
    plan = moe_b200.GroupedGemmPlan(2, device).from_ep_counts(torch.tensor([30, 10]), 1, 2)
    xq, wq = moe_b200.quantize_fp8(x), moe_b200.quantize_fp8_weight(w)
    assert torch.equal(moe_b200.grouped_gemm_fp8(xq, wq, plan=plan), moe_b200.grouped_gemm_fp8(xq, wq, [30, 10]))
