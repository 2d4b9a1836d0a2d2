"""Reading 8-bit rows back over the whole range of both types, and what of it bf16 can hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_every_value_and_scale(cuda_dev):
    """All 256 e4m3 bytes under all 256 scale bytes: the product, rounded once to bf16. That is exact but
    for results below 2^-133, bf16's smallest, and from 2^128 on, which are infinite."""
    import moe_b200
    codes = torch.arange(256, dtype=torch.uint8).view(1, 256).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat(1, 2)
    q = moe_b200.Fp8Tensor(codes.view(torch.float8_e4m3fn).to(cuda_dev), scales.view(torch.float8_e8m0fnu).to(cuda_dev))
    got = moe_b200.dequantize_fp8(q).cpu()
    value = codes.view(torch.float8_e4m3fn).double()
    exact = value * torch.where(scales[:, :1] == 255, torch.nan, torch.ldexp(torch.ones(256, 1, dtype=torch.float64),
                                                                             scales[:, :1].int() - 127))
    want = exact.float().to(torch.bfloat16)  # fp32 holds the product whole
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(nan=0.0, posinf=float("inf"), neginf=-float("inf")),
                       want.nan_to_num(nan=0.0, posinf=float("inf"), neginf=-float("inf")))
    held = (exact.abs() >= 2.0 ** -133) & (exact.abs() < 2.0 ** 128) | (exact == 0)
    whole = held & ((exact / 2.0 ** -133).frac() == 0)
    assert bool((got.double()[whole] == exact[whole]).all())


def test_largest_values(cuda_dev):
    """Values from 1.9375 * 2^127 on round to 2^128, which the pair of value and scale holds and bf16
    does not; those below come back to half a step."""
    import moe_b200
    top = 1.9375 * 2.0 ** 127
    x = torch.tensor([top, -top, 1.9296875 * 2.0 ** 127, 2.0 ** 127] + [0.0] * 12).view(1, 16).to(cuda_dev)
    for src in (x, x.to(torch.bfloat16)):
        q = moe_b200.quantize_fp8(src)
        assert int(q.scale.view(torch.uint8)) == 247
        assert q.data.float()[0, :4].tolist() == [256.0, -256.0, 240.0, 128.0]
        back = moe_b200.dequantize_fp8(q)[0].float()
        assert back[:4].tolist() == [float("inf"), -float("inf"), 1.875 * 2.0 ** 127, 2.0 ** 127]
