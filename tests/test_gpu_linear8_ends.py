"""The epilogues of nb_linear8 at the ends of fp32: infinities, NaN and values
next to the largest through every activation, in the forms for few rows and
in tiles, against the formulas in 64 bits."""
import math

import numpy as np
import pytest
import torch

from nativebit_amd import ops

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
ENDS = [math.inf, -math.inf, math.nan, 3e38, -3e38, 0.0]
ACTIVATIONS = [None, "silu", "gelu", "swiglu"]


def layer(books, N, K, dev):
    """All weights the first entry of their block."""
    index = torch.zeros(N * K, dtype=torch.uint8, device=dev)
    return ops.linear8_layout(ops.pack(index, 3), books.to(dev), N, K)


def formula(v, activation):
    """activation(v) as its definition in 64 bits."""
    def silu(z):
        return z / (1 + torch.exp(-z))
    if activation == "silu":
        return silu(v)
    if activation == "gelu":
        return v * (1 + torch.special.erf(v / math.sqrt(2))) / 2
    if activation == "swiglu":
        return silu(v[:, 0::2]) * v[:, 1::2]
    return v


def same(got, want, dtype):
    """Equal to the 64-bit values rounded once: each is 0, a NaN, an infinity or a
    value that no step rounds."""
    want = want.float().to(dtype).double()
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), (got, want)
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)), (got, want)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("M", [1, 3, 40, 300])
def test_biases(dev, M, activation, dtype):
    """Rows of zeros: the outputs are those of the bias; every pair of ends for the
    gated product."""
    K = 128
    bias = torch.tensor([e for a in ENDS for b in ENDS for e in (a, b)])
    N = bias.numel()
    w = layer(torch.ones(N * K // 128, 8), N, K, dev)
    x = ops.Rows8(torch.zeros(M, K, dtype=torch.int8, device=dev), torch.ones(M, device=dev))
    want = formula(bias.double().expand(M, N), activation)
    y = ops.linear8(x, w, bias=bias.to(dev), activation=activation, out_dtype=DT[dtype])
    same(y, want, DT[dtype])
    r = torch.ones(M, want.shape[1], dtype=DT[dtype], device=dev)
    y = ops.linear8(x, w, bias=bias.to(dev), activation=activation, residual=r)
    same(y, want + 1, DT[dtype])


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("M", [1, 40, 300])
def test_sums_past_fp32(dev, M, activation):
    """Scales whose product with the sums is over fp32: infinities of the sums' sign."""
    K, N = 256, 36
    books = torch.ones(N * K // 128, 8)
    books[::4] = books[1::4] = -1.0         # every other output
    w = layer(books, N, K, dev)
    x = ops.Rows8(torch.full((M, K), 127, dtype=torch.int8, device=dev), torch.full((M,), 1e38, device=dev))
    v = torch.full((M, N), math.inf, dtype=torch.float64)
    v[:, ::2] = -math.inf
    same(ops.linear8(x, w, activation=activation), formula(v, activation), torch.float32)


@pytest.mark.parametrize("far", [5.0, 14.0, 20.0])
@pytest.mark.parametrize("M", [1, 300])
def test_gelu_far_out(dev, M, far):
    """Where Phi is 1 to fp32's last bit, and where it falls below its range."""
    K, N = 128, 32
    bias = torch.linspace(-far, far, N)
    w = layer(torch.ones(N * K // 128, 8), N, K, dev)
    x = ops.Rows8(torch.zeros(M, K, dtype=torch.int8, device=dev), torch.ones(M, device=dev))
    y = ops.linear8(x, w, bias=bias.to(dev), activation="gelu").cpu().double()
    v = bias.double().numpy()
    want = torch.from_numpy(0.5 * v * torch.special.erfc(torch.from_numpy(-v / math.sqrt(2))).numpy())
    # Phi's tail: the exponent v^2 / 2 log2(e) with two roundings and a constant of half a step,
    # 1.5 steps of v^2 log2(e) ln 2 / 2 = v^2 / 2 each; the polynomial's eight steps, its
    # reciprocal, the exponential and three products: 16 steps; below 2^-126 nothing is asked for
    h = 2.0 ** -24
    tail = np.abs(v) * 0.5 * torch.special.erfc(torch.from_numpy(np.abs(v) / math.sqrt(2))).numpy()
    off = torch.from_numpy(tail * (2 * h) * (1.5 * v * v / 2 + 16) + h * np.abs(want.numpy()) + 2.0 ** -126)
    assert ((y - want).abs() <= off).all()
