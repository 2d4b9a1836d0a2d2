"""CPU checks of the 8-bit and group-router entry points: bad arguments are refused before any
device work, empty shapes are no-ops."""
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import moe_b200
    from moe_b200 import build
    build.build()
    return moe_b200.load_library()


def test_router_group_refusals(lib):
    f = lib.moe_router_group_topk

    def call(t=4, e=64, k=4, mode=2, groups=8, keep=2, gs=1, x=16, vals=16):
        return f(x, None, t, e, k, mode, groups, keep, gs, 1, 1.0, vals, None, None, None, None)
    assert call(e=60) == 1 and b"no multiple" in lib.moe_b200_last_error()
    assert call(groups=0) == 1
    assert call(mode=0) == 1
    assert call(gs=2) == 1
    assert call(keep=0) == 1 and call(keep=9) == 1
    assert call(k=0) == 1 and call(k=17) == 1  # 17 > 2 groups of 8
    assert call(k=17, keep=8) == 2  # valid, beyond this build
    assert call(e=2048, groups=8) == 2
    assert call(e=1024, groups=64) == 2
    assert call(vals=None) == 1 and b"no output" in lib.moe_b200_last_error()
    assert call(x=None) == 1
    assert call(t=0, x=None) == 0


def test_router_backward_refusals(lib):
    f = lib.moe_router_topk_backward

    def call(t=4, e=64, k=4, mode=1, gv=16, gp=None, x=16, out=16, idx=16):
        return f(x, None, None, idx, gv, gp, t, e, k, mode, 1, 1.0, out, None)
    assert call(mode=3) == 1 and call(mode=-1) == 1
    assert call(k=0) == 1 and call(k=33) == 1 and call(e=3) == 1
    assert call(gv=None) == 1 and call(gp=16) == 1
    assert b"exactly one" in lib.moe_b200_last_error()
    assert call(x=None) == 1 and call(out=None) == 1 and call(idx=None) == 1
    assert call(t=0, x=None, gv=None) == 0


def test_quantise_refusals(lib):
    q = lib.moe_quantize_fp8
    assert q(16, 2, 4, 64, 16, 16, None) == 1
    assert q(16, 0, 4, 24, 16, 16, None) == 1 and q(16, 0, 4, 0, 16, 16, None) == 1
    assert q(8, 0, 4, 64, 16, 16, None) == 1 and q(16, 0, 4, 64, 24, 16, None) == 1
    assert q(None, 0, 4, 64, 16, 16, None) == 1
    assert q(None, 0, 0, 64, None, None, None) == 0
    w = lib.moe_quantize_fp8_weight
    assert w(16, 0, 70000, 64, 64, 16, 16, None) == 1
    assert w(16, 0, 2, 0, 64, 16, 16, None) == 1 and w(16, 0, 2, 64, 40, 16, 16, None) == 1
    assert w(None, 0, 0, 64, 64, None, None, None) == 0
    d = lib.moe_dequantize_fp8
    assert d(16, 16, 4, 40, 16, None) == 1 and d(16, 16, 4, 64, 24, None) == 1
    assert d(None, None, 0, 64, None, None) == 0
    p = lib.moe_permute_fp8
    assert p(16, 16, 16, 33, 16, 16, 4, 64, 8, 32, None) == 1
    assert p(16, 16, 16, 0, 16, 16, 4, 64, 8, 32, None) == 1
    assert p(16, 16, 16, 4, 16, 16, 4, 40, 8, 32, None) == 1
    assert p(None, 16, 16, 4, 16, 16, 4, 64, 8, 32, None) == 1
    assert p(None, None, None, 4, None, None, 0, 64, 8, 0, None) == 0


def test_gemm_refusals(lib):
    f = lib.moe_grouped_gemm_fp8
    big = 1 << 20

    def call(x=256, xs=256, w=256, ws=256, out=256, osc=None, pre=None, rows=8, g=2, nw=2, n=256,
             k=256, kn=0, epi=0, wsp=256, wb=big):
        return f(x, xs, w, ws, out, osc, pre, rows, g, nw, n, k, kn, epi, wsp, wb, None)
    assert call(epi=2) == 1
    assert call(k=24) == 1 and call(k=0) == 1
    assert call(n=12) == 1 and call(n=24, kn=1) == 1
    assert call(epi=1, kn=1, osc=256) == 1
    assert call(epi=1, n=128, osc=256) == 1 and call(epi=1, n=384, osc=256) == 1
    assert call(epi=1) == 1 and b"out_scale" in lib.moe_b200_last_error()
    assert call(pre=256) == 1
    assert call(g=0) == 1 and call(nw=0) == 1 and call(rows=-1) == 1
    assert call(wsp=None) == 1 and call(wb=16) == 1 and call(wsp=128) == 1
    assert call(x=None) == 1 and call(xs=None) == 1 and call(ws=None) == 1
    assert call(x=264) == 1 and call(w=264) == 1 and call(out=264) == 1
    assert call(rows=0, x=None) == 0


def test_ops_refuse_cpu_tensors_and_bad_arguments():
    import moe_b200
    lg = torch.randn(4, 8)
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q = moe_b200.Fp8Tensor(torch.zeros(4, 64, dtype=torch.float8_e4m3fn),
                           torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu))
    for call in (lambda: moe_b200.router_group_topk(lg, 2),
                 lambda: moe_b200.router_topk_backward(lg, torch.zeros(4, 2, dtype=torch.int64),
                                                       grad_vals=torch.zeros(4, 2)),
                 lambda: moe_b200.quantize_fp8(x), lambda: moe_b200.quantize_fp8_weight(x[None]),
                 lambda: moe_b200.dequantize_fp8(q),
                 lambda: moe_b200.permute_fp8(x, torch.zeros(4, 8, dtype=torch.int64),
                                              torch.zeros(4, 2, dtype=torch.int64), 8),
                 lambda: moe_b200.grouped_gemm_fp8(q, q)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()


@pytest.mark.gpu
def test_ops_refuse_bad_shapes(cuda_dev):
    import moe_b200
    lg = torch.randn(4, 8, device=cuda_dev)
    ix = torch.zeros(4, 2, dtype=torch.int64, device=cuda_dev)
    gv = torch.zeros(4, 2, device=cuda_dev)
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda_dev)
    q = moe_b200.quantize_fp8(x)
    w = moe_b200.quantize_fp8_weight(torch.zeros(2, 24, 64, dtype=torch.bfloat16, device=cuda_dev))
    plan3 = moe_b200.GroupedGemmPlan(3, cuda_dev).from_splits(torch.tensor([1, 1, 2]))
    bad = [lambda: moe_b200.router_group_topk(lg, 2, num_groups=3),
           lambda: moe_b200.router_group_topk(lg, 9),
           lambda: moe_b200.router_group_topk(lg, 2, score="logits"),
           lambda: moe_b200.router_group_topk(lg, 2, group_score="sum"),
           lambda: moe_b200.router_group_topk(lg, 2, num_groups=2, topk_groups=3),
           lambda: moe_b200.router_group_topk(lg, 2, bias=gv[0]),
           lambda: moe_b200.router_group_topk(lg.double(), 2),
           lambda: moe_b200.router_topk_backward(lg, ix),
           lambda: moe_b200.router_topk_backward(lg, ix, grad_vals=gv, grad_probs=lg),
           lambda: moe_b200.router_topk_backward(lg, ix, grad_vals=lg),
           lambda: moe_b200.router_topk_backward(lg, ix.int(), grad_vals=gv),
           lambda: moe_b200.router_topk_backward(lg, ix, grad_vals=gv, score="tanh"),
           lambda: moe_b200.quantize_fp8(x[:, :24]), lambda: moe_b200.quantize_fp8(x.half()),
           lambda: moe_b200.quantize_fp8(x[0]), lambda: moe_b200.quantize_fp8_weight(x),
           lambda: moe_b200.dequantize_fp8(moe_b200.Fp8Tensor(q.data, q.scale[:2])),
           lambda: moe_b200.dequantize_fp8(moe_b200.Fp8Tensor(x, q.scale)),
           lambda: moe_b200.permute_fp8(x, ix, ix[:2], 4),
           lambda: moe_b200.permute_fp8(x, ix, ix, -1),
           lambda: moe_b200.grouped_gemm_fp8(q, w, plan=plan3),
           lambda: moe_b200.grouped_gemm_fp8(q, w, [1, 1, 2]),
           lambda: moe_b200.grouped_gemm_fp8(q, w, [3, 3]),
           lambda: moe_b200.grouped_gemm_fp8(q, w, epilogue="swiglu_fp8"),
           lambda: moe_b200.grouped_gemm_fp8(q, w, return_pre=True),
           lambda: moe_b200.grouped_gemm_fp8(q, w, w_layout="KN"),
           lambda: moe_b200.grouped_gemm_fp8(q, moe_b200.Fp8Tensor(w.data, w.scale[:, :0])),
           lambda: moe_b200.grouped_gemm_fp8(q, w, [-1, 5]),
           lambda: moe_b200.grouped_gemm_fp8(q, moe_b200.Fp8Tensor(w.data[:0], w.scale[:0])),
           lambda: moe_b200.grouped_gemm_fp8(q, w, epilogue="fp32")]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was not refused")
