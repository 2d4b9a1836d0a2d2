"""Gradient of renormalised routing weights where the scores are tiny, saturated or far apart: against
the formula in 64 bits, to the roundings that it meets."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32


def sigmoid_grad64(x, idx, g, renorm, scale):
    """(gradient of the taken logits [T,k], magnitude of its terms) in 64 bits: with w = s / sum s
    d/dx_j sum_i g_i w_i = w_j (1 - s_j) (g_j - sum_i g_i w_i); without renorm g_j s_j (1 - s_j).
    s from log-sigmoids, so that nothing underflows."""
    v = x.double().gather(1, idx)
    g = g.double() * scale
    ls = torch.nn.functional.logsigmoid(v)
    rest = torch.sigmoid(-v)
    if not renorm:
        return g * ls.exp() * rest, g.abs() * ls.exp() * rest
    w = torch.softmax(ls, 1)
    dot, mag = (g * w).sum(1, keepdim=True), (g.abs() * w).sum(1, keepdim=True)
    return w * rest * (g - dot), w * rest * (g.abs() + mag)


def case(t, e, k, low, high, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.rand(t, e, generator=gen) * (high - low) + low
    idx = torch.rand(t, e, generator=gen).argsort(1)[:, :k].contiguous()
    return x, idx, torch.randn(t, k, generator=gen)


def run(dev, x, idx, g, **kw):
    import moe_b200
    return moe_b200.router_topk_backward(x.to(dev), idx.to(dev), grad_vals=g.to(dev), **kw).cpu()


def check(got, idx, want, mag, steps):
    t, e = got.shape
    full = torch.zeros(t, e, dtype=torch.float64).scatter_(1, idx, want)
    room = torch.zeros(t, e, dtype=torch.float64).scatter_(1, idx, mag)
    assert bool(torch.isfinite(got).all())
    # 1e-43: a weight below fp32's normal numbers is off by its last bits, 2^-149 each
    err = (got.double() - full).abs() - 1e-43 * (1 + mag.amax())
    assert bool((err <= steps * U * room).all()), float((err / (U * room).clamp_min(1e-300)).max())


def test_smallest_example(cuda_dev):
    """Two logits near -60: s is about 1e-26, the square of their sum below fp32's range."""
    x, idx = torch.tensor([[-60.0, -60.5]]), torch.tensor([[0, 1]])
    got = run(cuda_dev, x, idx, torch.tensor([[1.0, 0.0]]), score="sigmoid", renorm=True)
    w = 1 / (1 + torch.exp(torch.tensor(-0.5, dtype=torch.float64)))  # of the first
    want = torch.stack([w * (1 - w), -w * (1 - w)])[None]
    assert bool(((got.double() - want).abs() <= 100 * U).all())


# Roundings of the renormalised form, in half steps: expf 4 (two ulp), 1 + e^-|v| 3, a quotient 1, the
# argument of the exponential as many as its size (|d| of a list's spread), a sum of k terms 5 (a tree); w
# meets two such exponentials' errors (22 + 2 d), sum g w of it 7 more, 1 - s 8, the last three operations 3:
# below 64 + 4 d of the terms' magnitude.
@pytest.mark.parametrize("low,high", [(-100.0, -40.0), (-45.5, -44.5), (-60.0, -59.0), (-81.0, -79.0), (-96.0, -94.0),
                                      (-300.0, -299.0), (-700.0, -699.0), (-4.0, 4.0), (5.0, 12.0), (14.0, 30.0),
                                      (60.0, 80.0), (-80.0, 80.0)])
@pytest.mark.parametrize("t,e,k", [(1, 8, 2), (67, 64, 8), (130, 256, 12), (65, 48, 20)])
def test_sigmoid_renormalised(cuda_dev, t, e, k, low, high):
    x, idx, g = case(t, e, k, low, high, t + int(high))
    got = run(cuda_dev, x, idx, g, score="sigmoid", renorm=True, scale=2.5)
    check(got, idx, *sigmoid_grad64(x, idx, g, True, 2.5), 64 + 4 * (high - low))


@pytest.mark.parametrize("low,high", [(-80.0, -40.0), (-4.0, 4.0), (5.0, 12.0), (14.0, 30.0), (60.0, 80.0)])
def test_sigmoid_plain(cuda_dev, low, high):
    """s (1 - s) without cancellation: two quotients of one exponential, 8 half steps each, and two
    products."""
    x, idx, g = case(65, 64, 8, low, high, 3)
    got = run(cuda_dev, x, idx, g, score="sigmoid", renorm=False, scale=2.5)
    check(got, idx, *sigmoid_grad64(x, idx, g, False, 2.5), 24)


def test_lists_whose_forward_weights_are_zero(cuda_dev):
    """Scores of logits below -709.78 are 0 in 64 bits, so the forward gives such lists zero weights:
    their gradient is 0; a list that holds one larger logit has its gradient."""
    import moe_b200
    x = torch.full((3, 16), -800.0)
    x[1] = -float("inf")
    x[2, 3] = -700.0
    dev = x.to(cuda_dev)
    r = moe_b200.router_group_topk(dev, 4, renorm=True)
    assert bool((r.topk_vals[:2] == 0).all()) and bool(r.topk_vals[2, 0] == 1)
    g = torch.randn(3, 4, generator=torch.Generator().manual_seed(1)).to(cuda_dev)
    got = moe_b200.router_topk_backward(dev, r.topk_idx, grad_vals=g, score="sigmoid", renorm=True)
    assert bool((got[:2] == 0).all()) and bool(torch.isfinite(got).all())


@pytest.mark.parametrize("size", [1e-30, 1e-22, 1.0, 1e22, 1e30])
@pytest.mark.parametrize("k", [2, 8, 20])
def test_logits_renormalised(cuda_dev, size, k):
    """Weights x_j / S of positive logits whose square leaves fp32's range:
    d/dx_j sum_i g_i w_i = (g_j - sum_i g_i w_i) / S. Sum 5 half steps, w 6, sum g w 13, the rest 3."""
    x, idx, g = case(50, 64, k, 0.5, 2.0, k)
    x = x * size
    got = run(cuda_dev, x, idx, g, score="logits", renorm=True)
    v, gd = x.double().gather(1, idx), g.double()
    S = v.sum(1, keepdim=True)
    w = v / S
    dot, mag = (gd * w).sum(1, keepdim=True), (gd.abs() * w).sum(1, keepdim=True)
    want, room = (gd - dot) / S, (gd.abs() + mag) / S
    check(got, idx, want, room, 32)


def test_gradient_against_differences(cuda_dev):
    """Of the forward itself, in 64 bits, at logits near -60."""
    x, idx, g = case(6, 12, 4, -61.0, -59.0, 2)
    got = run(cuda_dev, x, idx, g, score="sigmoid", renorm=True).double()
    step = 1e-4

    def value(v):
        s = torch.sigmoid(v).gather(1, idx)
        return (s / s.sum(1, keepdim=True) * g.double()).sum(1)
    for j in range(12):
        d = torch.zeros(6, 12, dtype=torch.float64)
        d[:, j] = step
        want = (value(x.double() + d) - value(x.double() - d)) / (2 * step)
        # the third derivative times step^2 / 6 is below 1e-7 here, and the kernel's roundings
        assert bool(((got[:, j] - want).abs() <= 1e-6 * (1 + want.abs())).all())
