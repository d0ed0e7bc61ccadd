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
