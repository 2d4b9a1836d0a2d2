"""Selection of the group-limited router where the fp32 pass has to leave it to 64 bits: scores a few
fp32 steps apart on either side of the border in rows of every width, and the shapes that are selected
in 64 bits throughout."""
import pytest
import torch

from test_gpu_router_ties import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e,k", [(64, 4), (256, 8), (384, 8), (512, 8), (1024, 8), (1024, 16)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("spread", [0.001, 0.1, 1.0, 6.0])
def test_border_within_the_bound(cuda_dev, e, k, score, spread):
    """The k-th and the next expert from 1 to 64 units of 2^-23 apart in their softmax scores
    (logits that differ by as much), in rows from flat to peaked, whose normaliser sums up E terms."""
    t = 16384
    g = torch.Generator(device=cuda_dev).manual_seed(e + k)
    x = torch.randn(t, e, generator=g, device=cuda_dev) * spread
    v, i = x.sort(dim=1, descending=True)
    steps = torch.randint(1, 65, (t, 1), generator=g, device=cuda_dev).float()
    x.scatter_(1, i[:, k:k + 1], v[:, k - 1:k] - steps * 2.0 ** -23)
    check(x, k, score, 1, 1)


@pytest.mark.parametrize("e,groups,keep,k", [(1023, 3, 2, 8), (1020, 5, 2, 8), (1017, 9, 4, 8), (1024, 1, 1, 8),
                                             (1020, 17, 6, 6), (1023, 31, 9, 5)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_wide_lanes(cuda_dev, e, groups, keep, k, score):
    """32 columns a lane and, where the groups leave lanes empty, more."""
    g = torch.Generator(device=cuda_dev).manual_seed(groups)
    x = torch.randn(3000, e, generator=g, device=cuda_dev)
    bias = torch.randn(e, generator=g, device=cuda_dev) * 0.05
    for logits in (x, (x * 8).round() / 8, x * 30):
        for b in (None, bias):
            for group_score in ("top2", "max"):
                check(logits, k, score, groups, keep, b, group_score)
