"""The widths on both sides of the borders between the second derivative's kernels, long and short structures together."""
import pytest
import torch

import test_structure_attention as base


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("width", [32, 33, 63, 64, 65, 66, 67, 112, 113, 128])
@pytest.mark.parametrize("lens", [[45, 7, 130], [200, 33] + [3] * 90])
def test_second_derivative_at_every_border(dtype, width, lens):
    base._run((lens, 2, 1, width, 0.1, 3), dtype, "cuda")
