"""Rows in 8 bits and their products at the largest numbers of rows: row tiles and
row ranges past 65535."""
import pytest
import torch

from nativebit_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [65535 * 16, 65535 * 16 + 1, 1 << 20])
def test_most_rows_of_few_outputs(dev, M):
    N, K = 16, 128
    g = torch.Generator().manual_seed(3)
    books = torch.randint(-127, 128, (N, 8), generator=g).float()
    books[:, 0] = 127.0                                                   # scales of 1
    index = torch.randint(0, 8, (N, K), generator=g, dtype=torch.uint8)
    w = ops.linear8_layout(ops.pack(index.reshape(-1).to(dev), 3), books.to(dev), N, K)
    x = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8).to(dev)
    scale = (2.0 ** torch.randint(-3, 4, (M,), generator=g)).to(dev)
    y = ops.linear8(ops.Rows8(x, scale), w)
    # whole numbers under 2^21 times powers of two: exact in fp32, in any order
    weights = torch.gather(books, 1, index.long())
    want = torch.matmul(x.float(), weights.T.contiguous().to(dev)) * scale[:, None]
    assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width", [(65535, 20), (65536, 33), (131071, 20)])
def test_values_of_many_rows(dev, rows, width, dtype):
    g = torch.Generator().manual_seed(4)
    codes = torch.randint(-127, 128, (rows, width), generator=g, dtype=torch.int8).to(dev)
    scale = torch.rand(rows, generator=g).to(dev)
    got = ops.Rows8(codes, scale).values(dtype)
    assert torch.equal(got, (codes.float() * scale[:, None]).to(dtype))
    x = torch.randn(rows, width, generator=g).to(dev)
    q = ops.quantize8(x)
    some = torch.tensor([0, 1, 65533, 65534, rows - 1], device=dev)
    few = ops.quantize8(x[some])
    assert torch.equal(q.codes[some], few.codes) and torch.equal(q.scale[some], few.scale)
