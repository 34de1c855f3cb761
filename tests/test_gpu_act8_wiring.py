"""TransformerBlock8's wiring on the GPU: which tensor each call of a block gets, to the
bit, with norm weights, layers and streams that all differ; its attention against 64
bits."""
import math

import pytest
import torch

from nativebit_amd import ops
from nativebit_amd.model import ModelConfig, init_kv_cache, quantize_activations, random_packed_model
from nativebit_amd.paged import PagedCache

pytestmark = pytest.mark.gpu
CFG = dict(vocab_size=300, n_layers=3, n_embd=256, n_head=4, ffn_hidden=384, context_len=64)


@pytest.fixture(scope="module")
def model(dev):
    m = random_packed_model(ModelConfig(**CFG), seed=7, device=dev)
    g = torch.Generator().manual_seed(8)
    with torch.no_grad():
        for norm in [n for b in m.blocks for n in (b.ln1, b.ln2)]:
            norm.weight.copy_(torch.rand(256, generator=g) + 0.5)
    for b in m.blocks:
        b.ln2.eps = 1e-3
    return quantize_activations(m)


@pytest.fixture
def calls(monkeypatch):
    """Every call of a norm, quantization and product: (name, arguments, result)."""
    seen = []

    def record(name):
        f = getattr(ops, name)

        def run(*args, **kw):
            got = f(*args, **kw)
            keep = [a.clone() if isinstance(a, torch.Tensor) else a for a in args]
            seen.append((name, keep, {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}, got))
            return got
        monkeypatch.setattr(ops, name, run)
    for name in ("rmsnorm8", "quantize8", "linear8"):
        record(name)
    return seen


def check_attention(qkv, att, cos, sin, heads):
    """att is the causal attention of the (B, T, 3 C) rows, adjacent pairs turned, in 64
    bits; the positions are 0 .. T - 1."""
    B, T, C = qkv.shape[0], qkv.shape[1], qkv.shape[2] // 3
    D = C // heads
    q, k, v = (t.reshape(B, T, heads, D).transpose(1, 2) for t in qkv.double().cpu().split(C, dim=-1))

    def turn(t):
        c, s = cos[:T].double().cpu(), sin[:T].double().cpu()
        even, odd = t[..., 0::2], t[..., 1::2]
        return torch.stack([even * c - odd * s, even * s + odd * c], -1).flatten(-2)
    q, k = turn(q), turn(k)
    products = q[..., :, None, :] * k[..., None, :, :] / math.sqrt(D)
    scores = products.sum(-1).masked_fill(torch.ones(T, T).triu(1).bool(), -math.inf)
    want = (scores.softmax(-1) @ v).transpose(1, 2).reshape(B, T, C)
    # fp32 half steps h.  A score is off by the sum's D steps and the turns' and scale's ten
    # of its products (turned pairs are as long as the pairs: their length stands for them);
    # a weight's exponential by that and 8, its sum by T; the mean by twice that (numerator
    # and denominator) and its own T + 4, of the largest value
    h = 2.0 ** -24
    pairs = (q.unflatten(-1, (-1, 2)).norm(dim=-1)[..., :, None, :] *
             k.unflatten(-1, (-1, 2)).norm(dim=-1)[..., None, :, :]).sum(-1).max().item() * 2 / math.sqrt(D)
    off = (2 * ((D + 10) * pairs + 8 + T) + T + 4) * h * v.abs().max().item()
    assert (att.reshape(B, T, C).double().cpu() - want).abs().max() <= off


def check_block(block, x, out, seen):
    """One block's eight calls: names, inputs, weights, results."""
    assert [c[0] for c in seen] == ["rmsnorm8", "linear8", "quantize8", "linear8", "rmsnorm8", "linear8",
                                    "quantize8", "linear8"]
    (_, a1, k1, h1), (_, a2, k2, qkv), (_, a3, k3, q3), (_, a4, k4, stream), (_, a5, k5, h5), (_, a6, k6, gated), \
        (_, a7, k7, q7), (_, a8, k8, last) = seen
    x = x.reshape(-1, 256)

    def norm(args, kw, rows, ln):
        assert not kw and torch.equal(args[0], rows) and torch.equal(args[1], ln.weight) and args[2] == ln.eps

    def product(args, kw, rows8, layer, activation, residual):
        assert args[0] is rows8
        assert args[1].tiles.data_ptr() == layer.tiles.data_ptr()
        assert args[1].scale.data_ptr() == layer.scale.data_ptr()
        assert kw["bias"] is None and kw["activation"] == activation and kw["out_dtype"] is None
        assert kw["residual"] is None if residual is None else torch.equal(kw["residual"], residual)
    norm(a1, k1, x, block.ln1)
    product(a2, k2, h1, block.attn.qkv, None, None)
    product(a4, k4, q3, block.attn.out_proj, None, x)
    norm(a5, k5, stream, block.ln2)
    product(a6, k6, h5, block.gate_up, "swiglu", None)
    assert torch.equal(a7[0], gated)
    product(a8, k8, q7, block.down, None, stream)
    assert torch.equal(out.reshape(-1, 256), last)
    return qkv, a3[0]                                    # attention's rows in and out


def outputs(model):
    """The blocks' inputs and outputs in a pass."""
    seen = []
    return seen, [b.register_forward_hook(lambda m, i, o: seen.append((i[0].clone(), o[0].clone())))
                  for b in model.blocks]


def run(model, f):
    seen, hooks = outputs(model)
    try:
        got = f()
    finally:
        for h in hooks:
            h.remove()
    return got, seen


@pytest.mark.parametrize("B,T", [(1, 1), (2, 19), (3, 64)])
def test_dense_pass(dev, model, calls, B, T):
    idx = torch.randint(0, 300, (B, T), generator=torch.Generator().manual_seed(T)).to(dev)
    (hidden, _), seen = run(model, lambda: model.hidden(idx))
    assert torch.equal(seen[0][0].reshape(B, T, 256), model.embedding.weight[idx].float())
    for i, b in enumerate(model.blocks):
        x, out = seen[i]
        if i:
            assert torch.equal(x, seen[i - 1][1])
        qkv, att = check_block(b, x, out, calls[8 * i:8 * i + 8])
        check_attention(qkv.view(B, T, 768), att, b.attn.cos, b.attn.sin, 4)
    assert len(calls) == 8 * len(model.blocks)


def test_cached_steps_are_the_dense_pass(dev, model, calls):
    """Step after step over the fp32 cache: each block's calls, positions moved on."""
    idx = torch.randint(0, 300, (1, 12), generator=torch.Generator().manual_seed(3)).to(dev)
    caches = init_kv_cache(model, 1, dev)
    rows = []
    for t in range(12):
        del calls[:]
        (_, caches), seen = run(model, lambda: model.hidden(idx[:, t:t + 1], caches, t))
        rows.append([check_block(b, *seen[i], calls[8 * i:8 * i + 8]) for i, b in enumerate(model.blocks)])
    for i, b in enumerate(model.blocks):
        qkv = torch.cat([r[i][0] for r in rows])
        att = torch.cat([r[i][1] for r in rows])
        check_attention(qkv.view(1, 12, 768), att, b.attn.cos, b.attn.sin, 4)


def test_paged_step(dev, model, calls):
    cache = PagedCache(model, 8, 2, device=dev)
    cache.step([5, 9])
    idx = torch.randint(0, 300, (1, 14), generator=torch.Generator().manual_seed(4)).to(dev)
    _, seen = run(model, lambda: model.hidden(idx, cache))
    for i, b in enumerate(model.blocks):
        check_block(b, *seen[i], calls[8 * i:8 * i + 8])
