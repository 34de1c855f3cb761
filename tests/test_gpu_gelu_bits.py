"""The bits of GELU in nb_linear8's epilogue: outputs of small values, each within the
half steps of fp32 that its formula takes."""
import math

import pytest
import torch

from nativebit_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 300])
@pytest.mark.parametrize("most", [0.5, 0.1, 1e-3])
def test_small_values(dev, M, most):
    N, K = 1 << 16, 128
    packed = ops.pack(torch.zeros(N * K, dtype=torch.uint8, device=dev), 3)
    w = ops.linear8_layout(packed, torch.ones(N, 8, device=dev), N, K)
    x = ops.Rows8(torch.zeros(M, K, dtype=torch.int8, device=dev), torch.ones(M, device=dev))
    bias = ((torch.rand(N, generator=torch.Generator().manual_seed(1)) * 2 - 1) * most).to(dev)
    y = ops.linear8(x, w, bias=bias, activation="gelu")
    assert torch.equal(y, y[:1].expand(M, N))
    v = bias.double()
    want = v * torch.special.erfc(-v / math.sqrt(2)) / 2
    # In half steps: u takes 5 (its product with 0.21, the sum, a reciprocal within two, the
    # product), of which u P'(u) / P(u) < 0.35 reach P up to 0.5; P's nine steps 2 (its terms
    # fall off with u <= 0.1); the exponential 2 and its argument's 2 times 0.125; their
    # product 1; the polynomial 0.25; so the tail 7.25, no more in the outputs (the tail is
    # at most half of them on the right), and their own 1
    off = 8.25 * 2.0 ** -24 * want.abs() + 2.0 ** -149
    assert ((y[0].double() - want).abs() <= off).all()
