"""PackedLinear8's residual without a GPU: its leading dimensions are x's."""
import pytest
import torch

from nativebit_amd import PackedLinear8, ops


@pytest.mark.parametrize("x,residual", [
    ((2, 3, 128), (3, 2, 16)), ((2, 3, 128), (6, 16)), ((2, 3, 128), (1, 6, 16)), ((6, 128), (2, 3, 16)),
    ((128,), (1, 16)), ((128,), ()), ((4, 128), (16,)), ((1, 128), (16,)), ((0, 128), (0, 2, 16))])
def test_other_leading_dimensions_are_refused(x, residual):
    layer = PackedLinear8(ops.Weights8(torch.zeros(896, dtype=torch.uint8), torch.zeros(16), 16, 128))
    with pytest.raises(ValueError, match="residual"):
        layer(torch.zeros(x), residual=torch.zeros(residual))
