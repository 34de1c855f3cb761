"""Drawn tokens and layers for rows in 8 bits without a GPU: what generate, the
layers and the model's conversion refuse on the host."""
import types

import pytest
import torch

from nativebit_amd import PackedLinear, PackedLinear8, paged
from nativebit_amd.model import PackedGPT, quantize_activations


def test_generate_refuses_draws():
    model = types.SimpleNamespace(embedding=types.SimpleNamespace(weight=torch.zeros(10, 4)),
                                  context_len=20)
    u = torch.zeros(2, 3)
    for kw in (dict(top_k=3), dict(top_p=0.5), dict(min_p=0.1), dict(u=u), dict(generator=torch.Generator())):
        with pytest.raises(ValueError, match="temperature"):
            paged.generate(model, [[1], [2, 3]], 3, **kw)
    with pytest.raises(ValueError, match="generator"):
        paged.generate(model, [[1], [2, 3]], 3, temperature=1.0, u=u, generator=torch.Generator())
    for bad in (u[:1], u[0], u[:, :2], u[..., None]):
        with pytest.raises(ValueError, match="u must"):
            paged.generate(model, [[1], [2, 3]], 3, temperature=1.0, u=bad)
    for k in (2.5, [1, 2.0]):
        with pytest.raises(ValueError, match="whole"):
            paged.generate(model, [[1], [2, 3]], 3, temperature=1.0, top_k=k)
    for kw in (dict(temperature=[1.0]), dict(top_k=[1, 2, 3]), dict(top_p=[[0.5, 0.5]]), dict(min_p=[])):
        with pytest.raises(ValueError, match="must be a number"):
            paged.generate(model, [[1], [2, 3]], 3, **{"temperature": 1.0, **kw})


@pytest.mark.parametrize("kw", [dict(bits=4, n=16), dict(bits=3, n=8, block=64), dict(bits=3, n=8, K=192)])
def test_layers_of_other_formats(kw):
    K, block, bits, n = kw.get("K", 256), kw.get("block", 128), kw["bits"], kw["n"]
    blocks = -(-4 * K // block)
    layer = PackedLinear(torch.zeros(blocks * block * bits // 8, dtype=torch.uint8), torch.zeros(blocks, n), 4, K,
                         block_size=block, bits=bits)
    with pytest.raises(ValueError, match="3 bits"):
        PackedLinear8.from_packed_linear(layer)
    with pytest.raises(ValueError, match="3 bits"):
        PackedLinear8.from_pairs(layer, layer)


def test_other_layers():
    with pytest.raises(ValueError, match="3 bits"):
        PackedLinear8.from_packed_linear(torch.nn.Linear(256, 4))
    model = PackedGPT(16, 1, 64, 1, 128, 32, torch.nn.Linear)
    with pytest.raises(ValueError, match="3 bits"):
        quantize_activations(model)
    # refused by the layout: it has no CPU form
    layer = PackedLinear(torch.zeros(4 * 96, dtype=torch.uint8), torch.zeros(8, 8), 4, 256)
    with pytest.raises(ValueError):
        PackedLinear8.from_packed_linear(layer)
