"""GPU: products and gradients by expert where the ends of the groups are out of order or out of range."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from piper_offload_b200 import _native_fp4 as nat
from piper_offload_b200 import fp4

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def device_status_clean(cuda_device):
    yield
    assert nat.device_status(cuda_device) == 0, "a bounded device wait timed out"


ENDS = [[40, 25, 90, 90, 60, 200], [200, 0, 0, 0, 0, 0], [-5, 30, -7, 300, 10, 250], [0, 0, 130, 20, 5, 131],
        [3, 150, 2, 149, 151, 1] + [7] * 25 + [20, 190, 12, 191] + [0] * 8, [10 * i for i in range(16)] * 2]


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("ends", ENDS, ids=lambda e: "_".join(map(str, e[:6])))
def test_ends_out_of_order_count_as_the_largest_before_them(ends, fmt, cuda_device):
    tokens, rows, cols = 200, 136, 160
    g = torch.Generator(cuda_device).manual_seed(3)
    dense = torch.randn((len(ends), rows, cols), generator=g, device=cuda_device).bfloat16()
    w = fp4.quantize_mxfp4(dense) if fmt == "mxfp4" else fp4.quantize_nvfp4(dense)
    x = torch.randn((tokens, cols), generator=g, device=cuda_device).bfloat16()
    dy = torch.randn((tokens, rows), generator=g, device=cuda_device).bfloat16()
    ordered = np.maximum.accumulate(np.clip(ends, 0, tokens))
    results = []
    for e in (ordered, ends):
        t = torch.tensor(np.asarray(e), dtype=torch.int32, device=cuda_device)
        # scratch and outputs come from memory that holds NaN codes
        junk = [torch.full((1 << n,), 255, dtype=torch.uint8, device=cuda_device) for n in (14, 15, 16, 17, 18, 19) for _ in range(8)]
        del junk
        results.append((fp4.grouped_linear_fp4(x, w, t), fp4.grouped_linear_fp4_grad_input(dy, w, t)))
    for got, want in zip(results[1], results[0]):
        assert want.isfinite().all() and torch.equal(got, want)
        assert not want[int(ordered[-1]):].any()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_ends_out_of_order_of_few_rows_by_many_experts(fmt, cuda_device):
    """The product quantises its tokens itself, and finds tiles in three lots of ends."""
    experts, tokens, rows, cols = 70, 100, 136, 160
    g = torch.Generator(cuda_device).manual_seed(5)
    dense = torch.randn((experts, rows, cols), generator=g, device=cuda_device).bfloat16()
    w = fp4.quantize_mxfp4(dense, swizzled=True) if fmt == "mxfp4" else fp4.quantize_nvfp4(dense)
    assert nat.linear_plan(fp4._matrix(w)[0], tokens).fused
    x = torch.randn((tokens, cols), generator=g, device=cuda_device).bfloat16()
    ends = np.arange(experts) + np.random.default_rng(6).integers(-12, 13, experts)
    ordered = np.maximum.accumulate(np.clip(ends, 0, tokens))
    results = []
    for e in (ordered, ends):
        junk = [torch.full((1 << n,), 255, dtype=torch.uint8, device=cuda_device) for n in range(14, 20) for _ in range(8)]
        del junk
        results.append(fp4.grouped_linear_fp4(x, w, torch.tensor(e, dtype=torch.int32, device=cuda_device)))
    assert results[0].isfinite().all() and torch.equal(*results)
    assert not results[0][int(ordered[-1]):].any() and results[0][:int(ordered[-1])].any(dim=1).all()
