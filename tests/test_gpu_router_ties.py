"""Selection of the group-limited router where scores are equal, or equal in fp32, inside the columns
of one lane: against a 64-bit restatement on the GPU, for every number of columns a lane can hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# E, groups, groups kept, k; columns a lane holds, which are consecutive
WIDTHS = [(32, 1, 1, 4, 1), (64, 1, 1, 6, 2), (128, 1, 1, 8, 4), (128, 16, 5, 8, 4), (256, 1, 1, 8, 8),
          (256, 8, 4, 8, 8), (300, 1, 1, 8, 10), (384, 1, 1, 8, 12), (384, 32, 7, 6, 12), (512, 1, 1, 8, 16),
          (512, 16, 4, 8, 16), (1024, 1, 1, 16, 32), (1024, 32, 3, 9, 32), (1023, 3, 2, 8, 43), (1020, 17, 5, 6, 60)]


def taken64(x, k, score, groups, keep, group_score, bias):
    """(experts [T,k], scores s [T,E]) by the definition, in 64 bits on x's device."""
    x = x.double()
    t, e = x.shape
    s = 1 / (1 + torch.exp(-x)) if score == "sigmoid" else torch.softmax(x, 1)
    c = s if bias is None else s + bias.double()
    if keep < groups:
        top = torch.sort(c.view(t, groups, -1), dim=2, descending=True).values
        rank = top[:, :, :2].sum(2) if group_score == "top2" else top[:, :, 0]
        best = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :keep]
        stays = torch.zeros(t, groups, dtype=torch.bool, device=x.device).scatter_(1, best, True)
        c = torch.where(stays.repeat_interleave(e // groups, 1), c, torch.full_like(c, -float("inf")))
    return torch.sort(c, dim=1, descending=True, stable=True).indices[:, :k], s


def check(x, k, score, groups, keep, bias=None, group_score="top2"):
    import moe_b200
    r = moe_b200.router_group_topk(x, k, score=score, num_groups=groups, topk_groups=keep, bias=bias,
                                   group_score=group_score, renorm=False)
    idx, s = taken64(x, k, score, groups, keep, group_score, bias)
    wrong = (r.topk_idx != idx).any(1)
    assert not bool(wrong.any()), \
        f"{int(wrong.sum())} of {x.shape[0]} rows, first {r.topk_idx[wrong][0].tolist()} for {idx[wrong][0].tolist()}"
    w = s.gather(1, idx)
    # a 64-bit weight rounded once: half a step, and what the 64-bit sums of two programs differ by
    assert bool(((r.topk_vals.double() - w).abs() <= w * (2.0 ** -24 + 1e-12) + 1e-45).all())
    assert torch.equal(r.routing_map, torch.zeros_like(r.routing_map).scatter_(1, idx, True))


def low_rows(t, e, seed):
    """Logits below -1, those of a row all different in fp32 sigmoid and softmax scores."""
    g = torch.Generator().manual_seed(seed)
    steps = torch.rand(t, e, generator=g).argsort(1)
    return -1.0 - steps.float() / e


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_smallest_example(cuda_dev, score):
    for head in ([3.0, 2.0, 2.0], [2.0, 2.0, 2.0], [2.0, 2.0, 3.0], [2.0, 3.0, 2.0]):
        x = low_rows(1, 256, 1)
        x[0, :3] = torch.tensor(head)
        check(x.to(cuda_dev), 3, score, 1, 1)


# values that the columns of one lane get, the rest of the row stays below
PATTERNS = {
    "a better one, two equal": [3.0, 2.0, 2.0],
    "three equal": [2.0, 2.0, 2.0],
    "four equal": [2.0, 2.0, 2.0, 2.0],
    "two pairs": [3.0, 3.0, 2.0, 2.0],
    "five, three of them equal": [4.0, 3.0, 2.0, 2.0, 2.0],
    "saturated": [20.0, 22.0, 21.0],  # sigmoid 1 in fp32, different in 64 bits
    "all of one fp32 score": [12.0, 12.0 + 2.0 ** -18, 12.0 - 2.0 ** -18, 12.0 + 2.0 ** -17],
}


@pytest.mark.parametrize("e,groups,keep,k,width", WIDTHS)
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_ties_inside_one_lane(cuda_dev, e, groups, keep, k, width, score):
    """Every pattern at random columns of a random lane, in random order, for every k that ends
    among or behind the equal ones."""
    size = e // groups
    t = 2048
    g = torch.Generator().manual_seed(e + groups)
    for i, values in enumerate(PATTERNS.values()):
        m = min(len(values), width)
        x = low_rows(t, e, i)
        first = torch.randint(0, (size + width - 1) // width, (t, 1), generator=g) * width
        base = torch.randint(0, groups, (t, 1), generator=g) * size
        # m different columns of the lane: the places of the smallest of random numbers
        free = torch.rand(t, width, generator=g)
        free[torch.arange(width)[None] + first >= size] = 2.0
        cols = base + first + free.argsort(1)[:, :m]
        room = (torch.arange(width)[None] + first < size).sum(1) >= m
        order = torch.rand(t, m, generator=g).argsort(1)
        vals = torch.tensor(values[:m])[order]
        rows = torch.arange(t)[:, None].expand(-1, m)
        x[rows[room], cols[room]] = vals[room]
        x = x.to(cuda_dev)
        for kk in sorted({2, 3, k} & set(range(1, k + 1))):
            check(x, kk, score, groups, keep)


@pytest.mark.parametrize("e,groups,keep,k,width", WIDTHS)
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("kind", ["bf16", "bf16 wide", "copies of 2", "copies of 4", "saturated", "fp16 with bias"])
def test_random_rows_with_ties(cuda_dev, e, groups, keep, k, width, score, kind):
    """16384 rows of logits in which equal scores are common."""
    t = 16384
    g = torch.Generator(device=cuda_dev).manual_seed(e * 7 + groups)
    x = torch.randn(t, e, generator=g, device=cuda_dev)
    bias = None
    if kind == "bf16":
        x = x.to(torch.bfloat16).float()
    elif kind == "bf16 wide":
        x = (x * 4).to(torch.bfloat16).float()
    elif kind.startswith("copies"):  # every expert next to its copies, as an upcycled layer starts
        n = int(kind[-1])
        x = x[:, :(e + n - 1) // n].repeat_interleave(n, 1)[:, :e].contiguous()
    elif kind == "saturated":
        x = torch.where(x > 1.5, 17.0 + x * 2, x)
        bias = torch.randint(-1, 2, (e,), generator=g, device=cuda_dev).float() * 0.25
    else:
        x = x.to(torch.float16).float()
        bias = torch.randint(-8, 9, (e,), generator=g, device=cuda_dev).float() / 64
    check(x, k, score, groups, keep, bias)
    check(x[:2048].contiguous(), k, score, groups, keep, bias, "max")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("low", [-float("inf"), torch.finfo(torch.float32).min])
def test_ties_among_masked_columns(cuda_dev, score, low):
    """Rows that keep two to ten experts of one lane, equal or not: the rest is masked, and k reaches
    into the masked ones, which are equal as well."""
    e, k = 256, 8
    t = 512
    g = torch.Generator().manual_seed(3)
    x = torch.full((t, e), low)
    for r in range(t):
        n = int(torch.randint(2, 11, (1,), generator=g))
        at = int(torch.randint(0, e - n, (1,), generator=g))
        x[r, at:at + n] = torch.randint(0, 3, (n,), generator=g).float()
    for groups, keep in ((1, 1), (8, 3)):
        check(x.to(cuda_dev), k, score, groups, keep)
