"""MoELayer with 8-bit experts and with the group-limited router: every stage of a run against its
64-bit definition on the stage's own inputs, forward and backward, and the router's gradient."""
import pytest
import torch

import fp8_ref as ref
from test_gpu_fp8 import _check_swiglu, _product64
from test_gpu_router_group import route64

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8  # half a step of bf16, relative


def _setup(dev, t, h, e, f, seed):
    import moe_b200
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, h, generator=g).to(torch.bfloat16).to(dev)
    lg = torch.randn(t, e, generator=g).to(dev)
    w1 = (torch.randn(e, 2 * f, h, generator=g) * 0.05).to(torch.bfloat16).to(dev)
    w2 = (torch.randn(e, h, f, generator=g) * 0.05).to(torch.bfloat16).to(dev)
    go = torch.randn(t, h, generator=g).to(torch.bfloat16).to(dev)
    return x, lg, moe_b200.MoEWeights(w1, w2), go


def _routing(dev, e, groups, seed=5):
    import moe_b200
    g = torch.Generator().manual_seed(seed)
    return moe_b200.Routing(num_groups=groups, topk_groups=max(1, groups // 2), scale=2.5,
                            balance_bias=(torch.randn(e, generator=g) * 0.1).to(dev))


def _near(got, y, s, k):
    tol = BF16 * y.abs() + (1 + BF16) * k * 2.0 ** -24 * s
    assert bool(((got.double() - y).abs() <= tol).all())


def _wgrad64(dy, x, splits):
    out, mag, at = [], [], 0
    for m in splits:
        a, b = dy[at:at + m].double(), x[at:at + m].double()
        out.append(a.t() @ b)
        mag.append(a.abs().t() @ b.abs())
        at += m
    return torch.stack(out), torch.stack(mag)


@pytest.mark.parametrize("t,h,e,f,k,groups", [(1, 128, 8, 128, 2, 4), (70, 272, 16, 128, 4, 4),
                                              (513, 512, 32, 256, 8, 8), (1200, 1024, 8, 384, 3, 1)])
def test_run_of_the_operators(cuda_dev, t, h, e, f, k, groups):
    import moe_b200
    x, lg, w, go = _setup(cuda_dev, t, h, e, f, t + h)
    wq = moe_b200.MoEWeightsFp8.from_weights(w)
    route = _routing(cuda_dev, e, groups)
    layer = moe_b200.MoELayer(wq, topk=k, routing=route)
    out, ctx = layer.forward(x, lg, save_for_backward=True)
    # the fused inference path gives the same bits
    assert torch.equal(out, layer(x, lg))
    r, rim = ctx["routing"], ctx["rim"]
    _, idx = route64(lg.cpu(), k, "sigmoid", groups, route.topk_groups, "top2",
                     route.balance_bias.cpu(), True, 2.5)
    assert torch.equal(r.topk_idx.cpu(), idx)
    splits = rim.counts.tolist()
    dst = rim.map_te.gather(1, r.topk_idx)
    q = moe_b200.quantize_fp8(x)
    for a, b in zip(ctx["xp"], q):
        assert torch.equal(ref.bytes_of(a)[dst], ref.bytes_of(b)[:, None].expand(-1, k, -1))
    _check_swiglu(ctx["h"], ctx["y1"], *_product64(ctx["xp"], wq.w1, splits, "NK"), h)
    _near(ctx["y"], *_product64(ctx["h"], wq.w2, splits, "NK"), f)
    rows = ctx["y"].double()[dst]  # [T,k,H]
    gates = r.topk_vals.double()[:, :, None]
    want, mag = (rows * gates).sum(1), (rows * gates).abs().sum(1)
    assert bool(((out.double() - want).abs() <= BF16 * want.abs() + (2 * k + 2) * 2.0 ** -24 * mag).all())

    # backward, another forward in between
    layer(x, torch.randn(t, e, generator=torch.Generator().manual_seed(1)).to(cuda_dev))
    gx, gp, dw1, dw2 = layer.backward(go, ctx)
    assert layer.plan.device_error() == 0
    dy2, gp_want = moe_b200.combine_backward(go, ctx["y"], rim.map_te, r.probs)
    assert torch.equal(gp, gp_want)
    hv = ref.values(ctx["h"].data, ref.bytes_of(ctx["h"].scale), True)
    xv = ref.values(ctx["xp"].data, ref.bytes_of(ctx["xp"].scale), True)
    _near(dw2, *_wgrad64(dy2, hv, splits), max(splits))
    dy2q = moe_b200.quantize_fp8(dy2)
    plan = moe_b200.GroupedGemmPlan(e, cuda_dev).from_splits(rim.counts)
    dh = moe_b200.grouped_gemm_fp8(dy2q, wq.w2, plan=plan, w_layout="KN")
    _near(dh, *_product64(dy2q, wq.w2, splits, "KN"), h)
    dy1 = moe_b200.swiglu_backward(ctx["y1"], dh)
    _near(dw1, *_wgrad64(dy1, xv, splits), max(splits))
    dy1q = moe_b200.quantize_fp8(dy1)
    dxp = moe_b200.grouped_gemm_fp8(dy1q, wq.w1, plan=plan, w_layout="KN")
    _near(dxp, *_product64(dy1q, wq.w1, splits, "KN"), 2 * f)
    rows = dxp.double()[dst]
    want, mag = rows.sum(1), rows.abs().sum(1)
    assert bool(((gx.double() - want).abs() <= BF16 * want.abs() + (k + 1) * 2.0 ** -24 * mag).all())


def test_near_the_bf16_layer(cuda_dev):
    """The 8-bit layer approximates the bf16 one: every quantised operand is off by at most 2^-4 of
    a value, on average about 2.6 %, and two products in a row meet four of them."""
    import moe_b200
    x, lg, w, go = _setup(cuda_dev, 300, 512, 16, 256, 3)
    a = moe_b200.MoELayer(w, topk=4)
    b = moe_b200.MoELayer(moe_b200.MoEWeightsFp8.from_weights(w), topk=4)
    oa, ca = a.forward(x, lg, save_for_backward=True)
    ob, cb = b.forward(x, lg, save_for_backward=True)
    assert torch.equal(ca["routing"].topk_idx, cb["routing"].topk_idx)
    pairs = [(oa, ob)] + list(zip(a.backward(go, ca), b.backward(go, cb)))
    for u, v in pairs:
        u, v = u.double(), v.double()
        assert float((u - v).norm() / u.norm()) < 0.15


@pytest.mark.parametrize("kind", ["softmax", "placed", "grouped", "gemm"])
def test_router_backward(cuda_dev, kind):
    """grad_logits of the layer against automatic differentiation of the gates in 64 bits."""
    import moe_b200
    t, h, e, f, k = 90, 256, 32, 128, 4
    x, lg, w, go = _setup(cuda_dev, t, h, e, f, 11)
    g = torch.Generator().manual_seed(2)
    bias = (torch.randn(e, generator=g) * 0.2).to(cuda_dev)
    perm = torch.randperm(e, generator=g).int().to(cuda_dev)
    kw = {"softmax": dict(expert_bias=bias), "placed": dict(expert_bias=bias, placement=perm),
          "grouped": dict(routing=_routing(cuda_dev, e, 4)), "gemm": dict(expert_bias=bias)}[kind]
    layer = moe_b200.MoELayer(w, topk=k, **kw)
    if kind == "gemm":  # the gate GEMM fused with the router
        rw = (torch.randn(e, h, generator=g) * 0.1).to(torch.bfloat16).to(cuda_dev)
        out, ctx = layer.forward(x, router_weight=rw, save_for_backward=True)
        assert torch.equal(out, layer(x, router_weight=rw))
        lg = ctx["logits"]
    else:
        out, ctx = layer.forward(x, lg, save_for_backward=True)
    gp = layer.backward(go, ctx)[1]
    got = layer.router_backward(gp, ctx).double()
    xd = lg.double().requires_grad_(True)
    idx = ctx["routing"].topk_idx
    cols = perm.long()[idx] if kind == "placed" else idx
    s = torch.sigmoid(xd) if kind == "grouped" else torch.softmax(xd + bias.double(), 1)
    wts = s.gather(1, cols)
    wts = wts / wts.sum(1, keepdim=True) * (2.5 if kind == "grouped" else 1.0)
    (wts * gp.double().gather(1, idx)).sum().backward()
    # terms that cancel: |g| and the mean of |g| under the weights, at most 64 roundings
    mag = 2.5 * 2 * gp.abs().amax(1, keepdim=True).double()
    assert bool(((got - xd.grad).abs() <= 64 * 2.0 ** -24 * mag).all())


def test_layer_refusals_and_empty(cuda_dev):
    import moe_b200
    from moe_b200.ep import MoELayerEP
    x, lg, w, go = _setup(cuda_dev, 4, 128, 8, 128, 1)
    with pytest.raises(ValueError):
        moe_b200.MoELayer(w, topk=2, routing=moe_b200.Routing(), expert_bias=lg[0].contiguous())
    _, _, odd, _ = _setup(cuda_dev, 4, 128, 8, 64, 1)
    with pytest.raises(ValueError):
        moe_b200.MoELayer(moe_b200.MoEWeightsFp8.from_weights(odd), topk=2)
    wq = moe_b200.MoEWeightsFp8.from_weights(w)
    with pytest.raises(ValueError):
        MoELayerEP(wq, num_experts=8)
    layer = moe_b200.MoELayer(wq, topk=2, routing=moe_b200.Routing(num_groups=2))
    assert layer(x[:0], lg[:0]).shape == (0, 128)
    out, ctx = layer.forward(x, lg, return_intermediates=True)
    with pytest.raises(ValueError):
        layer.backward(go, ctx)


def test_layer_in_a_graph_and_on_another_stream(cuda_dev):
    """Forward, backward and the router's gradient captured once and replayed on new inputs."""
    import moe_b200
    x, lg, w, go = _setup(cuda_dev, 200, 256, 16, 128, 7)
    wq = moe_b200.MoEWeightsFp8.from_weights(w)

    def step(layer):
        out, ctx = layer.forward(x, lg, save_for_backward=True)
        grads = layer.backward(go, ctx)
        return (out, *grads, layer.router_backward(grads[1], ctx))

    route = _routing(cuda_dev, 16, 4)
    layer, plain = (moe_b200.MoELayer(wq, topk=4, routing=route) for _ in range(2))
    step(layer)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(layer)
    side = torch.cuda.Stream()
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(200, 256, generator=g).to(torch.bfloat16))
        lg.copy_(torch.randn(200, 16, generator=g))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = step(plain)
        torch.cuda.synchronize()  # one training step at a time on a device (grouped_wgrad)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
