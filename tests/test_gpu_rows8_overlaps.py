"""Outputs given to the calls in 8 bits that overlap an input, on the GPU: refused, the
tensors left as they were."""
import pytest
import torch

from nativebit_amd import NativeBitError, ops

pytestmark = pytest.mark.gpu


def test_sum_over_the_weight(dev):
    room = torch.randn(5 * 64, device=dev)
    x, r = torch.randn(2, 4, 64, device=dev)
    keep = room.clone()
    for at in (0, 63, 64, 255, 256):
        weight = room[at:at + 64]
        with pytest.raises(ValueError, match="overlaps weight"):
            ops.rmsnorm8(x, weight, residual=r, out=room[:256].view(4, 64) if at < 256 else
                         room[4:260].view(4, 64))
    assert torch.equal(room, keep)
    weight = room[256:]
    rows8, total = ops.rmsnorm8(x, weight, residual=r, out=room[:256].view(4, 64))
    assert torch.equal(total, x + r) and torch.equal(weight, keep[256:])


def test_products_over_their_inputs(dev):
    N, K, M = 32, 128, 4
    room = torch.zeros(M * K + M * N * 4, dtype=torch.uint8, device=dev)
    codes = room[:M * K].view(torch.int8).view(M, K)
    packed = torch.zeros(N * K * 3 // 8, dtype=torch.uint8, device=dev)
    w = ops.linear8_layout(packed, torch.ones(N * K // 128, 8, device=dev), N, K)
    scale = torch.ones(M, device=dev)
    over = room[M * K - 128:M * K - 128 + M * N * 4].view(torch.float32).view(M, N)
    with pytest.raises(NativeBitError, match="overlap"):
        ops.linear8(ops.Rows8(codes, scale), w, out=over)
    bias = torch.zeros(M * N, device=dev)
    with pytest.raises(NativeBitError, match="overlap"):
        ops.linear8(ops.Rows8(codes, scale), w, bias=bias[:N], out=bias.view(M, N))
    beside = room[M * K:].view(torch.float32).view(M, N)
    assert ops.linear8(ops.Rows8(codes, scale), w, out=beside) is beside
