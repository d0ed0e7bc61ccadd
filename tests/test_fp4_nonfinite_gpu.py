"""GPU: two-level NVFP4 quantisation of matrices with values that are not finite, against the 64-bit definition."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import fp4_reference as R
from piper_offload_b200 import _native_fp4 as nat
from piper_offload_b200 import fp4

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def device_status_clean(cuda_device):
    yield
    assert nat.device_status(cuda_device) == 0, "a bounded device wait timed out"


def check_two_level(w, m: np.ndarray) -> None:
    """A two-level NVFP4 weight against its definition: the second level comes from the finite values, an infinity
    saturates its block's scale, a NaN marks its own block."""
    second = float(w.per_tensor_scale)
    assert second == R.second_of(np.where(np.isfinite(m), m, 0.0))
    codes, byte = R.quantize(m, "nvfp4", second=second)
    np.testing.assert_array_equal(w.scale.view(torch.uint8).cpu().numpy(), byte)
    known = np.repeat(byte != 127, 16, axis=1)
    np.testing.assert_array_equal(R.unpack(w.qdata.cpu().numpy())[known], codes[known])
    back = fp4.dequantize_fp4(w, torch.float32).double().cpu().numpy()
    assert np.isnan(back[~known]).all()
    # a product of a second level with the rest, rounded once
    np.testing.assert_allclose(back[known], R.values(codes, byte, "nvfp4", second)[known], rtol=2.0 ** -23)


@pytest.mark.parametrize("offset", [0, 1], ids=["aligned", "unaligned"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(5, 64), (40, 224), (300, 544), (1, 16)])
def test_second_level_of_a_matrix_with_values_that_are_not_finite(shape, dtype, offset, cuda_device):
    """Matrices on both sides of the size from which the maximum has a launch of its own."""
    rows, cols = shape
    base = np.random.default_rng([rows, cols]).standard_normal((rows, cols + offset)) * 0.02
    for bad in ((np.nan,), (np.inf,), (-np.inf,), (np.nan, -np.inf, np.inf)):
        x = torch.from_numpy(base).to(device=cuda_device, dtype=dtype)
        for i, v in enumerate(bad):
            x[(7 * i + 1) % rows, offset + (29 * i + 9) % cols] = v
        x = x[:, offset:]
        check_two_level(fp4.quantize_nvfp4(x), x.double().cpu().numpy())


def test_second_level_without_a_finite_value(cuda_device):
    for v in (float("nan"), float("inf")):
        x = torch.full((4, 32), v, device=cuda_device)
        w = fp4.quantize_nvfp4(x)
        assert float(w.per_tensor_scale) == 2.0 ** -23
        assert (w.scale.view(torch.uint8) == (127 if v != v else 126)).all()


@pytest.mark.parametrize("rows", [40, 1100])
def test_a_value_that_is_not_finite_stays_in_its_matrix_and_block(rows, cuda_device):
    x = torch.randn((3, rows, 96), generator=torch.Generator(cuda_device).manual_seed(2), device=cuda_device).bfloat16()
    clean = fp4.quantize_nvfp4(x)
    top = float(x[1].abs().max())
    x[1, 3, 20], x[1, 7, 40] = float("nan"), float("inf")
    assert float(x[1].nan_to_num(0, 0, 0).abs().max()) == top  # the replaced values were not the largest
    w = fp4.quantize_nvfp4(x)
    assert torch.equal(w.per_tensor_scale, clean.per_tensor_scale)
    same = w.qdata == clean.qdata
    same[1, 3, 8:16] = same[1, 7, 16:24] = True
    assert same.all()
    back = fp4.dequantize_fp4(w)
    assert back[1, 3, 16:32].isnan().all() and int(back.isnan().sum()) == 16
    # the largest code times the largest scale times the second level
    assert back[1, 7, 40] == (6 * 448 * w.per_tensor_scale[1]).bfloat16()
