"""Rows in 8 bits times packed layers with 8-bit codebooks on the GPU: the
layout byte for byte, products within the roundings of their fp32 epilogue."""
import numpy as np
import pytest
import torch

from nativebit_amd import ops
from nativebit_amd import pack as host_pack
from tests import rows8_ref as ref

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def layer(N, K, seed, dev):
    rng = np.random.default_rng(seed)
    index = rng.integers(0, 8, (N, K), dtype=np.uint8)
    books = np.sort(rng.standard_normal((N, K // 128, 8)) * 0.02 * rng.uniform(0.5, 2, (N, 1, 1)), -1)
    books = books.astype(np.float32)
    packed = ops.pack(torch.from_numpy(index.reshape(-1)).to(dev), 3)
    w = ops.linear8_layout(packed, torch.from_numpy(books.reshape(-1, 8)).to(dev), N, K)
    return index, books, w


def rows(M, K, seed):
    rng = np.random.default_rng(seed + 1)
    x = rng.integers(-127, 128, (M, K)).astype(np.int8)
    return x, (rng.uniform(0.001, 0.1, M)).astype(np.float32)


@pytest.mark.parametrize("N,K", [(1, 128), (16, 128), (17, 256), (40, 640), (100, 2560), (5, 6912)])
def test_layout(dev, N, K):
    index, books, w = layer(N, K, N + K, dev)
    q, scale = ref.layer8(books)
    assert np.array_equal(w.scale.cpu().numpy(), scale)
    assert np.array_equal(w.tiles.cpu().numpy(), ref.tiles(index, q))


def test_layout_of_outputs_that_are_zero_or_not_finite(dev):
    index, books, _ = layer(20, 256, 3, dev)
    books[4] = 0
    books[7, 1, 3] = np.nan
    books[18, 0, 0] = -np.inf
    w = ops.linear8_layout(ops.pack(torch.from_numpy(index.reshape(-1)).to(dev), 3),
                           torch.from_numpy(books.reshape(-1, 8)).to(dev), 20, 256)
    q, scale = ref.layer8(books)
    assert np.array_equal(w.scale.cpu().numpy(), scale, equal_nan=True)
    assert np.array_equal(w.tiles.cpu().numpy(), ref.tiles(index, q))
    x, xs = rows(3, 256, 5)
    y = ops.linear8(ops.Rows8(torch.from_numpy(x).to(dev), torch.from_numpy(xs).to(dev)), w).cpu()
    assert y[:, [7, 18]].isnan().all() and (y[:, 4] == 0).all()
    assert y.isnan().sum() == 6


def check(dev, M, N, K, dtype, bias=False, activation=None, residual=False, seed=0, w=None):
    index, books, w = w or layer(N, K, seed, dev)
    q, scale = ref.layer8(books)
    x, xs = rows(M, K, seed)
    rng = np.random.default_rng(seed + 2)
    out = N // 2 if activation == "swiglu" else N
    b = (rng.standard_normal(N) * 0.3).astype(np.float32) if bias else None
    r = torch.from_numpy(rng.standard_normal((M, out)).astype(np.float32)).to(DT[dtype]) if residual else None
    want, off = ref.linear8(x, xs, index, q, scale, b, activation,
                            None if r is None else r.float().numpy(), DT[dtype], dev)
    rows8 = ops.Rows8(torch.from_numpy(x).to(dev), torch.from_numpy(xs).to(dev))
    kw = dict(bias=None if b is None else torch.from_numpy(b).to(dev), activation=activation,
              residual=None if r is None else r.to(dev), out_dtype=DT[dtype])
    y = ops.linear8(rows8, w, **kw)
    assert y.dtype == DT[dtype] and y.shape == (M, out)
    bad = np.abs(y.double().cpu().numpy() - want) > off
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4])
    assert torch.equal(y, ops.linear8(rows8, w, **kw))      # (the same bits again)
    return rows8, w, kw, y


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 63, 64, 65, 129, 300, 513])
@pytest.mark.parametrize("N,K", [(1, 128), (33, 256), (130, 640), (257, 2560)])
def test_rows(dev, M, N, K):
    check(dev, M, N, K, "fp32", seed=M)


@pytest.mark.parametrize("N,K", [(2560, 2560), (7680, 2560), (2560, 6912), (1000, 128 * 64),
                                 (4, 1 << 17)])
@pytest.mark.parametrize("M", [1, 7, 40, 200])
def test_layers(dev, M, N, K):
    if N * K * M > 3e9:
        M = 24
    check(dev, M, N, K, "fp32", seed=N + M)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("activation", [None, "silu", "gelu", "swiglu"])
def test_epilogues(dev, activation, residual, bias, dtype):
    for M, N, K in ((1, 34, 256), (20, 70, 128), (150, 258, 384), (300, 518, 256)):
        check(dev, M, N, K, dtype, bias, activation, residual, seed=M)


# (rows, outputs, K) where each form of the product is the fastest, with whole and
# uneven shares of K, and rows and outputs that end inside its tiles
FORMS = [(2, 11, 256), (1, 14, 896), (1, 4110, 128), (2, 4099, 256), (1, 4104, 1152),          # rows
         (1, 12291, 384), (65, 8363, 256), (65, 8261, 640), (17, 8206, 1408),                  # 64 x 32
         (1, 8199, 128), (33, 8474, 384), (33, 12344, 896),                                    # 64 x 64
         (65, 10907, 256), (65, 10977, 1152),                                                  # 128 x 64
         (65, 8198, 128), (129, 10935, 256), (129, 11078, 640),
         (1024, 2560, 2560), (385, 14049, 1152),                                               # 128 x 128
         (518, 14693, 128), (517, 14490, 256), (516, 14875, 384)]                              # 256 x 256


@pytest.mark.parametrize("M,N,K", FORMS)
def test_forms(dev, M, N, K):
    w = layer(N, K, 5, dev)
    check(dev, M, N, K, "fp32", seed=5, w=w)
    check(dev, M, N, K, "bf16", True, "silu", True, seed=5, w=w)
    check(dev, M, N, K, "fp32", True, "gelu", seed=5, w=w)
    if N % 2 == 0:
        check(dev, M, N, K, "fp32", True, "swiglu", True, seed=5, w=w)
        check(dev, M, N, K, "bf16", False, "swiglu", seed=5, w=w)


def test_largest_sums(dev):
    """Codes of +-127 at the longest K: sums near 2^31."""
    N, K = 16, 1 << 17
    books = torch.zeros(N * K // 128, 8, device=dev)
    books[:, 0], books[:, 7] = -1.0, 1.0
    index = torch.full((N, K), 7, dtype=torch.uint8, device=dev)
    index[3] = 0
    w = ops.linear8_layout(ops.pack(index.reshape(-1), 3), books, N, K)
    for M in (1, 70, 300):
        x = torch.full((M, K), 127, dtype=torch.int8, device=dev)
        y = ops.linear8(ops.Rows8(x, torch.ones(M, device=dev)), w).double().cpu()
        want = torch.full((M, N), 127.0 * 127 * K / 127, dtype=torch.float64)
        want[:, 3] *= -1
        assert ((y - want).abs() <= 3.01 * 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("M", [1, 40, 300])
def test_strides_and_in_place(dev, M):
    N, K = 130, 512
    for dtype in DT:
        rows8, w, kw, y = check(dev, M, N, K, dtype, True, "silu", True, seed=9)
        # codes with a row stride, and misaligned ones (copied)
        wide = torch.zeros(M, K + 64, dtype=torch.int8, device=dev)
        wide[:, :K] = rows8.codes
        assert torch.equal(y, ops.linear8(ops.Rows8(wide[:, :K], rows8.scale), w, **kw))
        wide[:, 1:K + 1] = rows8.codes
        assert torch.equal(y, ops.linear8(ops.Rows8(wide[:, 1:K + 1], rows8.scale), w, **kw))
        # outputs and residual as columns of wider arrays; nothing around them changes
        big = torch.full((M + 2, N + 9), 5.0, dtype=DT[dtype], device=dev)
        big[1:M + 1, 3:N + 3] = kw["residual"]
        view = big[1:M + 1, 3:N + 3]
        got = ops.linear8(rows8, w, bias=kw["bias"], activation="silu", residual=view, out=view)
        assert got is view and torch.equal(view, y)
        assert (big[0] == 5).all() and (big[M + 1] == 5).all()
        assert (big[:, :3] == 5).all() and (big[:, N + 3:] == 5).all()


def test_no_rows(dev):
    _, _, w = layer(20, 128, 0, dev)
    y = ops.linear8(ops.Rows8(torch.empty(0, 128, dtype=torch.int8, device=dev),
                              torch.empty(0, device=dev)), w)
    assert y.shape == (0, 20)


def test_rows_whose_scale_is_nan(dev):
    _, _, w = layer(40, 256, 1, dev)
    x = torch.randn(20, 256, generator=torch.Generator().manual_seed(1))
    x[7, 3] = float("inf")
    y = ops.linear8(ops.quantize8(x.to(dev)), w).cpu()
    assert y[7].isnan().all() and not y[[i for i in range(20) if i != 7]].isnan().any()
