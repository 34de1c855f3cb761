"""quantize_activations without a GPU (the layout replaced by one that makes empty
tiles): a model is changed whole or not at all."""
import pytest
import torch

from nativebit_amd import ops
from nativebit_amd.linear import PackedLinear, PackedLinear8
from nativebit_amd.model import PackedGPT, TransformerBlock, TransformerBlock8, quantize_activations


def packed(out_features, in_features):
    n = out_features * in_features
    return PackedLinear(torch.zeros(n * 3 // 8, dtype=torch.uint8), torch.zeros(n // 128, 8),
                        out_features, in_features)


@pytest.fixture
def model(monkeypatch):
    def layout(packed, codebook, N, K):
        if N > 1 << 24 or K > 1 << 17:
            raise ValueError("too large")
        return ops.Weights8(torch.zeros((N + 15) // 16 * K * 7, dtype=torch.uint8), torch.zeros(N), N, K)
    monkeypatch.setattr(ops, "linear8_layout", layout)
    return PackedGPT(16, 3, 128, 2, 256, 32, packed)


def names(model):
    return {name: type(m) for name, m in model.named_modules()}


def test_all_blocks(model):
    attn = [b.attn for b in model.blocks]
    assert quantize_activations(model) is model
    for b, a in zip(model.blocks, attn):
        assert isinstance(b, TransformerBlock8) and b.attn is a
        assert all(isinstance(m, PackedLinear8) for m in (a.qkv, a.out_proj, b.gate_up, b.down))
        assert (b.gate_up.out_features, b.gate_up.in_features) == (512, 128)
    before = names(model)
    assert quantize_activations(model) is model and names(model) == before


@pytest.mark.parametrize("block", [0, 1, 2])
@pytest.mark.parametrize("wrong", ["pair", "layout", "format"])
def test_layers_that_do_not_fit_leave_the_model(model, block, wrong):
    ffn = model.blocks[block].ffn
    if wrong == "pair":
        ffn.up = packed(384, 128)                    # another size than the gate's
    elif wrong == "layout":
        ffn.down = packed(1, (1 << 17) + 128)        # more inputs than the products take
    else:
        ffn.down = torch.nn.Linear(256, 128)
    before = names(model)
    with pytest.raises(ValueError):
        quantize_activations(model)
    assert names(model) == before
    assert all(isinstance(b, TransformerBlock) for b in model.blocks)


def test_a_block_that_is_used_twice(model):
    model.blocks[2] = model.blocks[0]
    quantize_activations(model)
    assert model.blocks[0] is model.blocks[2] and isinstance(model.blocks[0], TransformerBlock8)
    assert isinstance(model.blocks[0].attn.qkv, PackedLinear8)
