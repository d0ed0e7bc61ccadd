"""GPU: groups that count by their two best experts, where the sums that decide are small beside what they are made of."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_routing_gpu import check_route, rng, to_torch

pytestmark = pytest.mark.gpu

# experts and groups: a lane's one, two, four and eight experts in groups that fill lanes, and groups that do not
SHAPES = [(16, 4), (64, 8), (96, 6), (128, 4), (256, 8), (12, 4), (512, 16)]


@pytest.mark.parametrize("offset", [0.0, 100.0, -1000.0, 1000.0, 30000.0])
@pytest.mark.parametrize("experts,groups", SHAPES)
def test_logits_far_from_zero(experts, groups, offset, cuda_device):
    """What a softmax adds to all logits changes nothing, so a group's sum may not lose bits of the logits. Spreads of some
    steps of the logits, at which many groups are next to each other."""
    step = float(np.spacing(np.float32(max(1.0, abs(offset)))))
    for spread in (0.3, 40 * step):
        logits = to_torch(offset + spread * rng(21, experts, groups).standard_normal((400, experts)), torch.float32, cuda_device)
        check_route(logits, groups // 2, groups=groups, top_groups=groups // 2, group_score="top2")


@pytest.mark.parametrize("alike", [True, False], ids=["alike", "apart"])
@pytest.mark.parametrize("size", [64.0, 1000.0, 1e5])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups", SHAPES)
def test_biases_that_cancel(experts, groups, scoring, size, alike, cuda_device):
    """Biases of one size and opposite signs in every group, or of another size in each: a group's sum is the scores' alone,
    of which neither part has more than a few bits."""
    per = experts // groups
    bias = np.repeat(-size * (np.ones(groups) if alike else 1 + np.arange(groups)), per).astype(np.float32)
    one = rng(22, experts).integers(0, per, groups) + np.arange(groups) * per
    bias[one] *= -1
    for dtype, spread in ((torch.float32, 0.02), (torch.float32, 1.0), (torch.bfloat16, 0.3)):
        logits = to_torch(spread * rng(23, experts, groups).standard_normal((200, experts)), dtype, cuda_device)
        check_route(logits, groups // 2, scoring=scoring, bias=bias, groups=groups, top_groups=groups // 2, group_score="top2")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups", SHAPES)
def test_biases_at_the_ends_of_the_range(experts, groups, scoring, cuda_device):
    """Sums that are infinite in fp32, or not a number, and groups that are closed in part or as a whole."""
    g = rng(24, experts)
    for values in ([3e38, -3e38, 0.0], [3.4e38, 3.3e38, -3.4e38], [np.inf, -np.inf, 1.0], [np.nan, 0.0, 1e30], [-np.inf, -3.4e38, 0.1]):
        bias = g.choice(np.array(values, np.float32), experts)
        logits = to_torch(g.standard_normal((60, experts)), torch.float32, cuda_device)
        for group_score in ("top2", "max"):
            check_route(logits, groups // 2, scoring=scoring, bias=bias, groups=groups, top_groups=groups // 2, group_score=group_score)
