"""Rows in 8 bits on the GPU (quantize8, rmsnorm8) against 64 bits: codes and
sums bit for bit, scales within their rounding."""
import numpy as np
import pytest
import torch

from nativebit_amd import ops
from tests import rows8_ref as ref

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
SIZES = [(1, 1), (1, 3), (2, 4), (1, 128), (5, 129), (3, 1023), (3, 1024), (3, 1025), (2, 2560),
         (4, 4096), (4, 4097), (2, 6912), (2, 8191), (2, 8192), (2, 8193), (1, 20001), (700, 640)]


def rows(n, width, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, width, generator=g) * (torch.rand(n, 1, generator=g) * 5 + 0.1)
    if n > 1:
        x[1] = 0          # a row of zeros
    return x.to(dtype)


def strided(x, dev, pad):
    """x on the GPU as columns of a wider array, one element in."""
    if not pad:
        return x.to(dev), None
    wide = torch.full((x.shape[0], x.shape[1] + pad), 7.0, dtype=x.dtype, device=dev)
    wide[:, 1:1 + x.shape[1]] = x.to(dev)
    return wide[:, 1:1 + x.shape[1]], wide


def check(got, q, scale):
    assert np.array_equal(got.codes.cpu().numpy(), q)
    # (64 bits rounded once: at most the neighbour where sums round differently)
    s = got.scale.cpu().numpy()
    assert np.array_equal(np.isnan(s), np.isnan(scale))
    assert (np.abs(s - scale) <= 2.0 ** -24 * 1.0001 * np.abs(scale) + 1e-45)[~np.isnan(s)].all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,width", SIZES)
def test_quantize8(dev, n, width, dtype):
    x = rows(n, width, DT[dtype], n + width)
    for pad in (0, 3):
        xd, wide = strided(x, dev, pad)
        q, scale = ref.quantize8(x)
        got = ops.quantize8(xd)
        check(got, q, scale)
        assert np.array_equal(got.scale.cpu().numpy(), scale)   # (a / 127 rounds once)
        values = torch.from_numpy(q.astype(np.float32)) * torch.from_numpy(scale)[:, None]
        assert torch.equal(got.values().cpu(), values)
        assert torch.equal(got.values(torch.bfloat16).cpu(), values.to(torch.bfloat16))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n,width", SIZES)
def test_rmsnorm8(dev, n, width, dtype):
    x = rows(n, width, DT[dtype], n + width + 1)
    r = rows(n, width, DT[dtype], n + width + 2).flip(0)
    w = torch.randn(width, generator=torch.Generator().manual_seed(3)) * 0.3 + 1
    wd = w.to(dev)
    for pad in (0, 2):
        xd, _ = strided(x, dev, pad)
        rd, _ = strided(r, dev, 2 * pad)
        q, scale, _ = ref.rmsnorm8(x, w, 1e-6)
        check(ops.rmsnorm8(xd, wd), q, scale)
        q, scale, h = ref.rmsnorm8(x, w, 1e-5, r)
        got, total = ops.rmsnorm8(xd, wd, 1e-5, residual=rd)
        check(got, q, scale)
        assert torch.equal(total.cpu(), h)
        # in place, on x and on the residual
        keep = rd.clone()
        got, total = ops.rmsnorm8(xd, wd, 1e-5, residual=rd, out=rd)
        check(got, q, scale)
        assert total is rd and torch.equal(rd.cpu(), h)
        got, total = ops.rmsnorm8(xd, wd, 1e-5, residual=keep, out=xd)
        check(got, q, scale)
        assert torch.equal(xd.cpu(), h)


@pytest.mark.parametrize("width", [5, 2560, 9000])
def test_not_finite(dev, width):
    """A NaN or an infinity is its own row's alone: scale NaN, codes 0."""
    x = rows(6, width, torch.float32, 4)
    x[0, width // 2] = float("nan")
    x[2, 0] = float("inf")
    x[3, width - 1] = -float("inf")
    x[4, :] = 1e38           # (squares past fp32)
    x[5, :] = 1e-38
    q, scale = ref.quantize8(x)
    got = ops.quantize8(x.to(dev))
    check(got, q, scale)
    assert np.isnan(scale[[0, 2, 3]]).all() and not np.isnan(scale[[1, 4, 5]]).any()
    w = torch.ones(width)
    q, scale, _ = ref.rmsnorm8(x, w, 1e-6)
    check(ops.rmsnorm8(x.to(dev), w.to(dev)), q, scale)


def test_ties_go_to_even(dev):
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5]])
    got = ops.quantize8(x.to(dev))
    assert got.codes[0].tolist() == [127, 0, 2, 2, 0, -2, -2, 126] and got.scale.item() == 1.0


def test_eps_and_a_row_of_zeros(dev):
    x = torch.zeros(2, 300)
    x[1, 7] = 1e-12
    w = torch.ones(300)
    for eps in (0.0, 1e-6):
        q, scale, _ = ref.rmsnorm8(x, w, eps)
        check(ops.rmsnorm8(x.to(dev), w.to(dev), eps), q, scale)


def test_no_rows(dev):
    for got in (ops.quantize8(torch.empty(0, 5, device=dev)),
                ops.rmsnorm8(torch.empty(0, 5, device=dev), torch.ones(5, device=dev))):
        assert got.codes.shape == (0, 5) and got.scale.shape == (0,)
