"""GPU parity of the group-limited router and of the gradient of routing weights, against plain
64-bit restatements."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _scores(x, score):
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    m = x.amax(1, keepdim=True)
    p = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(x), torch.exp(x - m))
    z = p.sum(1, keepdim=True)
    return torch.where(z == 0, torch.zeros_like(p), p / z)


def route64(logits, k, score, groups, keep, group_score, bias, renorm, scale):
    """(weights [T,k], idx [T,k]) by the definition, in 64 bits on the CPU."""
    x = logits.double()
    t, e = x.shape
    s = _scores(x, score)
    c = s if bias is None else s + bias.double()
    top = torch.sort(c.view(t, groups, -1), dim=2, descending=True).values
    rank = top[:, :, :2].sum(2) if group_score == "top2" else top[:, :, 0]
    kept = torch.zeros(t, groups, dtype=torch.bool)
    kept.scatter_(1, torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :keep], True)
    kept = kept.repeat_interleave(e // groups, 1)
    order = torch.sort(c, dim=1, descending=True, stable=True).indices
    inside = torch.sort(kept.gather(1, order).int(), dim=1, descending=True, stable=True).indices
    idx = order.gather(1, inside)[:, :k]
    return weights64(s, idx, renorm, scale), idx


def weights64(s, idx, renorm, scale):
    w = s.gather(1, idx)
    if renorm:
        total = w.sum(1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / total)
    return w * scale


def _check(r, w, idx, e):
    assert torch.equal(r.topk_idx.cpu(), idx)
    # the 64-bit weight rounded once: half a step, 2^-24, and the 64-bit arithmetic's own 1e-12
    got = r.topk_vals.cpu().double()
    assert bool(((got - w).abs() <= w.abs() * (2.0 ** -24 + 1e-12) + 1e-45).all())
    on = torch.zeros(idx.shape[0], e, dtype=torch.bool).scatter_(1, idx, True)
    assert torch.equal(r.routing_map.cpu(), on)
    assert torch.equal(r.probs.cpu(), torch.zeros(idx.shape[0], e).scatter_(1, idx, r.topk_vals.cpu()))


SHAPES = [  # T, E, k, groups, keep
    (1, 1, 1, 1, 1), (1, 8, 2, 2, 1), (5, 12, 3, 4, 2), (33, 64, 8, 8, 3), (7, 160, 6, 8, 3),
    (300, 256, 8, 8, 4), (129, 256, 16, 1, 1), (64, 320, 8, 32, 5), (9, 1024, 8, 16, 2),
    (50, 60, 4, 1, 1), (21, 40, 5, 5, 1), (16, 32, 16, 32, 16), (2, 2, 2, 1, 1)]


@pytest.mark.parametrize("t,e,k,groups,keep", SHAPES)
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("group_score", ["top2", "max"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route(cuda_dev, t, e, k, groups, keep, score, group_score, with_bias):
    import moe_b200
    g = torch.Generator().manual_seed(t + e + k)
    x = torch.randn(t, e, generator=g) * 2
    bias = torch.randn(e, generator=g) * 0.1 if with_bias else None
    renorm, scale = (t + e) % 2 == 0, 2.5
    r = moe_b200.router_group_topk(x.to(cuda_dev), k, score=score, num_groups=groups, topk_groups=keep,
                                   group_score=group_score, renorm=renorm, scale=scale,
                                   bias=None if bias is None else bias.to(cuda_dev))
    _check(r, *route64(x, k, score, groups, keep, group_score, bias, renorm, scale), e)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_route_ties_and_near_ties(cuda_dev, score):
    """Equal scores go to the lower expert and group; scores that differ by less than fp32 shows
    are told apart."""
    import moe_b200
    t, e, k = 64, 64, 8
    g = torch.Generator().manual_seed(3)
    cases = [torch.zeros(t, e), torch.randint(0, 3, (t, e), generator=g).float(),
             torch.full((t, e), 60.0), torch.full((t, e), -60.0)]
    near = torch.full((t, e), 0.5)
    near += torch.randint(0, 4, (t, e), generator=g) * 2.0 ** -24  # one step of 0.5 apart
    cases.append(near)
    big = 12.0 + torch.randint(0, 8, (t, e), generator=g) * 2.0 ** -20  # sigmoid moves by 2^-37
    cases.append(big)
    for bias in (None, torch.randint(0, 2, (e,), generator=g).float() * 2.0 ** -25):
        for x in cases:
            r = moe_b200.router_group_topk(x.to(cuda_dev), k, score=score, num_groups=8, topk_groups=3,
                                           bias=None if bias is None else bias.to(cuda_dev))
            _check(r, *route64(x, k, score, 8, 3, "top2", bias, True, 1.0), e)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_masked_logits(cuda_dev, score, renorm):
    """-inf and the type's lowest value as masks, rows that keep fewer than k experts or none."""
    import moe_b200
    t, e, k = 40, 32, 4
    g = torch.Generator().manual_seed(8)
    for low in (-float("inf"), torch.finfo(torch.float32).min):
        x = torch.randn(t, e, generator=g)
        x[torch.rand(t, e, generator=g) < 0.8] = low
        x[0], x[1, 1:], x[2, :-1] = low, low, low
        x[3] = 1.0
        r = moe_b200.router_group_topk(x.to(cuda_dev), k, score=score, num_groups=4, topk_groups=2,
                                       renorm=renorm)
        w, idx = route64(x, k, score, 4, 2, "top2", None, renorm, 1.0)
        _check(r, w, idx, e)
        assert bool(torch.isfinite(r.probs).all())


@pytest.mark.parametrize("e,groups,keep,k", [(128, 1, 1, 4), (128, 16, 5, 8), (256, 8, 4, 8), (384, 1, 1, 8),
                                             (384, 32, 7, 6), (512, 16, 4, 8), (1024, 1, 1, 16), (1024, 32, 3, 9),
                                             (1020, 17, 5, 6)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_route_wide_rows(cuda_dev, e, groups, keep, k, score):
    """Every layout of a row over the lanes: ties, near ties, masked logits, a bias that bars experts,
    unaligned rows."""
    import moe_b200
    t = 48
    g = torch.Generator().manual_seed(e + groups)
    x = torch.randn(t, e, generator=g) * 3
    ties = torch.randint(0, 40, (t, e), generator=g).float() / 8
    near = 1.0 + torch.randint(0, 64, (t, e), generator=g) * 2.0 ** -23
    masked = torch.where(torch.rand(t, e, generator=g) < 0.97, torch.full((t, e), -float("inf")), x)
    far = x * 40  # saturated and vanishing scores
    bar = torch.where(torch.rand(e, generator=g) < 0.3, torch.full((e,), -float("inf")), torch.zeros(e))
    small = torch.randint(-2, 3, (e,), generator=g).float() * 2.0 ** -6
    store = torch.empty(t * e + 1, device=cuda_dev)
    for logits in (x, ties, near, masked, far):
        for bias in (None, bar, small):
            for view in (logits.to(cuda_dev), store[1:].view(t, e).copy_(logits)):
                r = moe_b200.router_group_topk(view, k, score=score, num_groups=groups, topk_groups=keep,
                                               bias=None if bias is None else bias.to(cuda_dev), scale=0.5)
                _check(r, *route64(logits, k, score, groups, keep, "top2", bias, True, 0.5), e)


def test_route_nan_row_stays_in_its_row(cuda_dev):
    import moe_b200
    x = torch.randn(6, 32, generator=torch.Generator().manual_seed(1))
    x[2, 5] = float("nan")
    r = moe_b200.router_group_topk(x.to(cuda_dev), 4, num_groups=4, topk_groups=2)
    good = [0, 1, 3, 4, 5]
    w, idx = route64(x[good], 4, "sigmoid", 4, 2, "top2", None, True, 1.0)
    assert torch.equal(r.topk_idx.cpu()[good], idx)
    assert int(r.topk_idx[2, 0]) == 5 and bool(torch.isnan(r.topk_vals[2]).any())
    assert int(r.routing_map[2].sum()) == 4


def test_route_views_empty_and_maps_only(cuda_dev):
    import moe_b200
    x = torch.randn(64, 200, generator=torch.Generator().manual_seed(2)).to(cuda_dev)
    for v in (x[:, 1:129], x.t()[:, :32], x[3:20, 40:168]):
        r = moe_b200.router_group_topk(v, 4, num_groups=4, topk_groups=2, outputs="maps")
        full = moe_b200.router_group_topk(v.contiguous().clone(), 4, num_groups=4, topk_groups=2)
        assert r.topk_vals is None and torch.equal(r.routing_map, full.routing_map)
        assert torch.equal(r.probs, full.probs)
    r = moe_b200.router_group_topk(x[:0], 4, num_groups=4, topk_groups=2)
    assert r.probs.shape == (0, 200) and r.topk_idx.shape == (0, 4)


# ---------------------------------------------------------------------------------------- backward
def _weights_of(x, idx, score, renorm, scale, bias):
    x = x if bias is None else x + bias
    s = x if score == "logits" else torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, 1)
    w = s.gather(1, idx)
    return (w / w.sum(1, keepdim=True) if renorm else w) * scale


def _bwd_case(t, e, k, seed, positive):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, e, generator=g) * 2
    if positive:  # raw-logit weights: their sum must not come near zero
        x = x.abs() + 0.5
    idx = torch.rand(t, e, generator=g).argsort(1)[:, :k].contiguous()
    return x, idx, torch.randn(t, k, generator=g)


@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (3, 8, 2), (65, 160, 6), (200, 256, 8), (7, 64, 32), (5, 1500, 3),
                                   (37, 50, 12), (9, 20, 16)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax", "logits"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("dense", [False, True])
def test_backward(cuda_dev, t, e, k, score, renorm, dense):
    import moe_b200
    x, idx, gv = _bwd_case(t, e, k, t + e, score == "logits")
    bias = torch.randn(e, generator=torch.Generator().manual_seed(e)) * 0.3 if dense and score != "logits" else None
    xd = x.double().requires_grad_(True)
    bd = None if bias is None else bias.double()
    w = _weights_of(xd, idx, score, renorm, 2.5, bd)
    (w * gv.double()).sum().backward()
    want = xd.grad
    kw = {"grad_vals": gv.to(cuda_dev)}
    if dense:
        kw = {"grad_probs": torch.zeros(t, e).scatter_(1, idx, gv).to(cuda_dev)}
    got = moe_b200.router_topk_backward(x.to(cuda_dev), idx.to(cuda_dev), score=score, renorm=renorm,
                                        scale=2.5, bias=None if bias is None else bias.to(cuda_dev),
                                        **kw).cpu().double()
    # magnitude of the terms that cancel, and the roundings they meet: expf (2), sum, quotients and
    # products (at most 16), a sum of E/32 + 5 terms for the softmax normaliser, of k for the dots;
    # logits + bias is rounded too, an error of 2^-24 |x| in the exponent
    s = _weights_of(x.double(), idx, score, False, 1.0, bd).abs()
    S = s.sum(1, keepdim=True) if renorm else 1.0
    term = 2.5 * (gv.double().abs() / S + ((gv.double().abs() * s).sum(1, keepdim=True) / S / S if renorm else 0))
    full = x.double() if bd is None else x.double() + bd
    if score == "softmax":
        p = torch.softmax(full, 1)
        mag = p * (torch.zeros(t, e, dtype=torch.float64).scatter_(1, idx, term) + (term * s).sum(1, keepdim=True))
    elif score == "sigmoid":
        mag = torch.zeros(t, e, dtype=torch.float64).scatter_(1, idx, term * s)
    else:
        mag = torch.zeros(t, e, dtype=torch.float64).scatter_(1, idx, term)
    n = 18 + e / 32 + 5 + 2 * k + 4 * full.abs().amax()
    assert bool(((got - want).abs() <= n * 2.0 ** -24 * mag + 1e-40).all()), \
        float(((got - want).abs() / (2.0 ** -24 * mag).clamp_min(1e-300)).max())


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_backward_against_differences(cuda_dev, score):
    import moe_b200
    t, e, k = 6, 24, 4
    x, idx, gv = _bwd_case(t, e, k, 5, False)
    got = moe_b200.router_topk_backward(x.to(cuda_dev), idx.to(cuda_dev), grad_vals=gv.to(cuda_dev),
                                        score=score, renorm=True, scale=1.5).cpu().double()
    step = 1e-4
    want = torch.zeros(t, e, dtype=torch.float64)
    for j in range(e):
        d = torch.zeros(t, e, dtype=torch.float64)
        d[:, j] = step
        up = _weights_of(x.double() + d, idx, score, True, 1.5, None)
        dn = _weights_of(x.double() - d, idx, score, True, 1.5, None)
        want[:, j] = ((up - dn) * gv.double()).sum(1) / (2 * step)
    # central differences: the third derivative times step^2 / 6, below 1e-7 here, and fp32 roundings
    assert bool(((got - want).abs() <= 1e-6 * (1 + want.abs())).all())


def test_backward_masked_rows_bad_and_repeated_indices(cuda_dev):
    import moe_b200
    t, e, k = 8, 16, 3
    x, idx, gv = _bwd_case(t, e, k, 6, False)
    x[0] = -float("inf")
    x[1, :] = -float("inf")
    x[1, 4] = 0.5
    idx[1] = torch.tensor([4, 0, 1])
    for score in ("sigmoid", "softmax"):
        got = moe_b200.router_topk_backward(x.to(cuda_dev), idx.to(cuda_dev), grad_vals=gv.to(cuda_dev),
                                            score=score, renorm=True).cpu()
        assert bool(torch.isfinite(got).all()) and bool((got[0] == 0).all())
    # an index outside [0,E) takes no part; a repeated one gets the sum
    idx2 = idx.clone()
    idx2[3, 1], idx2[4, 0], idx2[5, 2] = -1, e, idx2[5, 0]
    got = moe_b200.router_topk_backward(x.to(cuda_dev), idx2.to(cuda_dev), grad_vals=gv.to(cuda_dev),
                                        score="sigmoid", renorm=False).cpu().double()
    s = torch.sigmoid(x.double())
    want = torch.zeros(t, e, dtype=torch.float64)
    for r in range(t):
        for j in range(k):
            c = int(idx2[r, j])
            if 0 <= c < e:
                want[r, c] += float(gv[r, j]) * float(s[r, c] * (1 - s[r, c]))
    assert bool(((got - want).abs() <= 32 * 2.0 ** -24 * (want.abs() + gv.abs().sum(1, keepdim=True))).all())


def test_backward_placement(cuda_dev):
    """Slots of a placed router: the gradient of model expert placement[c] from slot c."""
    import moe_b200
    t, e, k = 20, 16, 4
    g = torch.Generator().manual_seed(4)
    x = torch.randn(t, e, generator=g).to(cuda_dev)
    bias = (torch.randn(e, generator=g) * 0.2).to(cuda_dev)
    pl = torch.randperm(e, generator=g).int().to(cuda_dev)
    gp = torch.randn(t, e, generator=g).to(cuda_dev)
    r = moe_b200.router_topk(x, k, bias=bias, placement=pl)
    got = moe_b200.router_topk_backward(x, r.topk_idx, grad_probs=gp, bias=bias, placement=pl)
    perm = pl.long()
    want = moe_b200.router_topk_backward(x[:, perm].contiguous(), r.topk_idx, grad_probs=gp,
                                         bias=bias[perm].contiguous())
    assert torch.equal(got[:, perm], want)


@pytest.mark.parametrize("score,renorm", [("sigmoid", True), ("softmax", False), ("softmax", True)])
def test_backward_placement_out_of_range(cuda_dev, score, renorm):
    """A slot whose placement names no expert is one that the list does not name."""
    import moe_b200
    t, e, k = 5, 8, 3
    x, idx, gv = (v.to(cuda_dev) for v in _bwd_case(t, e, k, 9, False))
    pl = torch.arange(e, dtype=torch.int32, device=cuda_dev)
    pl[2], pl[5] = -1, e + 100
    kw = dict(grad_vals=gv, score=score, renorm=renorm)
    got = moe_b200.router_topk_backward(x, idx, placement=pl, **kw)
    gone = (idx == 2) | (idx == 5)
    assert bool(gone.any())
    want = moe_b200.router_topk_backward(x, torch.where(gone, torch.full_like(idx, -1), idx), **kw)
    assert torch.equal(got, want)


def test_router_in_a_graph(cuda_dev):
    import moe_b200
    x = torch.randn(100, 64, device=cuda_dev)
    gv = torch.randn(100, 4, device=cuda_dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = moe_b200.router_group_topk(x, 4, num_groups=8, topk_groups=2)
        d = moe_b200.router_topk_backward(x, r.topk_idx, grad_vals=gv, score="sigmoid")
    for seed in (1, 2):
        x.copy_(torch.randn(100, 64, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        e = moe_b200.router_group_topk(x, 4, num_groups=8, topk_groups=2)
        assert torch.equal(r.topk_idx, e.topk_idx) and torch.equal(r.probs, e.probs)
        assert torch.equal(d, moe_b200.router_topk_backward(x, e.topk_idx, grad_vals=gv, score="sigmoid"))
