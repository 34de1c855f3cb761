"""A model with its activations in 8 bits, and drawn tokens, on the GPU:
every norm, quantization, product and draw of its steps against 64 bits;
batches against requests one by one; captured and replayed steps."""
import numpy as np
import pytest
import torch

from nativebit_amd import ops, paged
from nativebit_amd import pack as host_pack
from nativebit_amd.decode import DecodeEngine
from nativebit_amd.linear import PackedLinear, PackedLinear8
from nativebit_amd.model import (ModelConfig, TransformerBlock8, greedy_generate, quantize_activations,
                                 random_packed_model, to_nbpack_params)
from tests import rows8_ref as ref

pytestmark = pytest.mark.gpu
CFG = dict(vocab_size=300, n_layers=2, n_embd=256, n_head=4, ffn_hidden=384, context_len=400)


def indices(layer):
    N, K = layer.out_features, layer.in_features
    return host_pack.unpack_nbits(layer.packed_indices.cpu(), N * K, 3).numpy().reshape(N, K).astype(np.uint8)


def parts(layer):
    """(indices, 8-bit codes, scale) of a packed layer."""
    books = layer.codebook.cpu().numpy().reshape(layer.out_features, -1, 8)
    return indices(layer), *ref.layer8(books)


def woven(a, b):
    return np.stack([a, b], 1).reshape(2 * a.shape[0], *a.shape[1:])


@pytest.fixture(scope="module")
def model(dev):
    """The model in 8 bits, and its layers' parts by their tiles' address."""
    m = random_packed_model(ModelConfig(**CFG), seed=5, device=dev)
    layers = [[parts(b.attn.qkv), parts(b.attn.out_proj),
               tuple(woven(x, y) for x, y in zip(parts(b.ffn.gate), parts(b.ffn.up))), parts(b.ffn.down)]
              for b in m.blocks]
    assert quantize_activations(m) is m and quantize_activations(m) is m
    m.parts = {}
    for b, of in zip(m.blocks, layers):
        assert isinstance(b, TransformerBlock8)
        for layer, p in zip((b.attn.qkv, b.attn.out_proj, b.gate_up, b.down), of):
            m.parts[layer.tiles.data_ptr()] = p
    return m


def checked(monkeypatch, model):
    """Every call of the four operators checked against the plain forms."""
    seen = []
    quantize8, rmsnorm8, linear8, sample = ops.quantize8, ops.rmsnorm8, ops.linear8, ops.sample

    def q8(x):
        got = quantize8(x)
        codes, scale = ref.quantize8(x.cpu())
        assert np.array_equal(got.codes.cpu().numpy(), codes)
        assert np.array_equal(got.scale.cpu().numpy(), scale)
        seen.append("quantize8")
        return got

    def n8(x, weight, eps=1e-6):
        got = rmsnorm8(x, weight, eps)
        codes, scale, _ = ref.rmsnorm8(x.cpu(), weight.cpu(), eps)
        assert np.array_equal(got.codes.cpu().numpy(), codes)
        # half a step of fp32, and the 64-bit sum's order
        assert (np.abs(got.scale.cpu().numpy() - scale) <= 2.0 ** -24 * 1.0001 * scale).all()
        seen.append("rmsnorm8")
        return got

    def l8(x, weights, *, bias=None, activation=None, residual=None, out_dtype=None):
        got = linear8(x, weights, bias=bias, activation=activation, residual=residual, out_dtype=out_dtype)
        index, q, scale = model.parts[weights.tiles.data_ptr()]
        want, off = ref.linear8(x.codes.cpu().numpy(), x.scale.cpu().numpy(), index, q, scale, None, activation,
                                None if residual is None else residual.cpu().numpy(), torch.float32)
        assert (np.abs(got.cpu().numpy() - want) <= off).all()
        seen.append("linear8")
        return got

    def draw(logits, u, **rules):
        got = sample(logits, u, **rules)
        rules = {name: t.cpu().tolist() for name, t in rules.items() if t is not None}
        for i, t in enumerate(got.tolist()):
            assert t == ref.sample(logits[i].cpu(), float(u[i]), **{n: r[i] for n, r in rules.items()})[0]
        seen.append("sample")
        return got
    for f in ((q8, "quantize8"), (n8, "rmsnorm8"), (l8, "linear8"), (draw, "sample")):
        monkeypatch.setattr(ops, f[1], f[0])
    return seen


BLOCK = ["rmsnorm8", "linear8", "quantize8", "linear8", "rmsnorm8", "linear8", "quantize8", "linear8"]
PROMPTS = [[7] * 70, [1, 2, 3], [299]]


def test_generate_draws(dev, model, monkeypatch):
    seen = checked(monkeypatch, model)
    u = torch.rand(3, 6, generator=torch.Generator().manual_seed(3))
    rules = dict(temperature=[0.7, 1.3, 0.0], top_k=[40, 0, 5], top_p=0.9, min_p=0.01)
    out = paged.generate(model, PROMPTS, 6, u=u, repetition=1.2, **rules)
    assert seen == 6 * (2 * BLOCK + ["sample"])
    assert [len(o) for o in out] == [6, 6, 6] and all(0 <= t < 300 for o in out for t in o)
    # a row's products, norms and attention do not depend on the others
    for i, p in enumerate(PROMPTS):
        own = {k: v[i] if isinstance(v, list) else v for k, v in rules.items()}
        assert paged.generate(model, [p], 6, u=u[i:i + 1], repetition=1.2, **own) == [out[i]]


def test_generate_draws_by_a_generator(dev, model):
    u = torch.rand(4, 3, generator=torch.Generator(dev).manual_seed(9), device=dev).t()
    want = paged.generate(model, PROMPTS, 4, u=u, temperature=1.0)
    assert paged.generate(model, PROMPTS, 4, generator=torch.Generator(dev).manual_seed(9),
                          temperature=1.0) == want
    assert len(paged.generate(model, PROMPTS, 4, temperature=1.0)) == 3
    # no random part: the first of the order, as without a temperature
    assert paged.generate(model, PROMPTS, 4, temperature=0.0) == paged.generate(model, PROMPTS, 4)
    assert paged.generate(model, PROMPTS, 4, temperature=5.0, top_k=1) == paged.generate(model, PROMPTS, 4)


def test_rows_that_the_mask_leaves_empty(dev, model):
    mask = torch.full((3, 10), -1, dtype=torch.int32, device=dev)
    mask[1] = 0
    out = paged.generate(model, PROMPTS, 3, temperature=0.8, mask=mask)
    assert out[1] == [-1, -1, -1] and min(out[0] + out[2]) >= 0


def test_caches_and_dense_forward(dev, model, monkeypatch):
    """The fp32 caches' step after step, and the pass without a cache."""
    seen = checked(monkeypatch, model)
    tokens = greedy_generate(model, [5, 6, 7], 4, device=dev)
    assert len(tokens) >= 4 and seen[:16] == 2 * BLOCK
    logits = model(torch.tensor([[5, 6, 7], [8, 9, 10]], device=dev))
    assert logits.shape == (2, 3, 300) and torch.isfinite(logits).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(256,), (1, 256), (2, 3, 256), (0, 256), (40, 256)])
def test_layer_near_the_exact_one(dev, dtype, shape):
    """Within what the roundings to 8 bits of inputs and entries can do."""
    m = random_packed_model(ModelConfig(**CFG), seed=6, device=dev)
    packed = m.blocks[0].ffn.gate
    layer = PackedLinear8.from_packed_linear(packed)
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    y = layer(x.to(dev)).cpu().double()
    assert y.shape == (*shape[:-1], 384) and layer(x.to(dev), out_dtype=dtype).dtype == dtype
    w = np.take_along_axis(packed.codebook.cpu().numpy().reshape(384, 2, 8).astype(np.float64),
                           indices(packed).reshape(384, 2, 128).astype(np.int64), 2).reshape(384, 256)
    w, x = torch.from_numpy(w), x.double()
    a = torch.from_numpy(np.abs(packed.codebook.cpu().numpy().reshape(384, 16)).max(1)).double()
    # half a step of 1/127 of the largest each, and the fp32 roundings of scales and outputs
    # (under 6 half steps of the products of the rounded)
    hx, hw = x.abs().amax(-1, keepdim=True) / 254, a / 254
    off = x.abs().sum(-1, keepdim=True) * hw + hx * w.abs().sum(1) + 256 * hx * hw
    top = (x.abs() + hx) @ (w.abs() + hw[:, None]).T
    assert ((y - x @ w.T).abs() <= off + 6 * 2.0 ** -24 * top).all()


def test_layer_takes_residual_and_bias(dev, model):
    m = random_packed_model(ModelConfig(**CFG), seed=6, device=dev)
    packed = m.blocks[0].ffn.down                                          # 256 x 384
    bias = torch.randn(256, generator=torch.Generator().manual_seed(2)).to(dev)
    layer = PackedLinear8.from_packed_linear(packed, bias)
    x, r = torch.randn(2, 5, 384, device=dev), torch.randn(2, 5, 256, device=dev)
    got = layer(x, activation="gelu", residual=r)
    plain = layer(x, activation="gelu")
    assert got.shape == (2, 5, 256) and torch.equal(got, plain + r)
    assert torch.equal(layer(ops.quantize8(x.view(10, 384)), activation="gelu"), plain.view(10, 256))
    # its buffers are its state
    again = PackedLinear8.from_packed_linear(m.blocks[1].ffn.down, torch.zeros_like(bias))
    again.load_state_dict(layer.state_dict())
    assert torch.equal(again(x, activation="gelu"), plain)


def test_captured_step(dev, model):
    """A step in a graph, replayed between eager steps of the same shapes: the
    eager step's results each time; two graphs of the same operators do not
    meet in a workspace."""
    g = torch.Generator().manual_seed(4)
    w = model.blocks[0].gate_up

    def step(x, r, u):
        h, s = ops.rmsnorm8(x, ones, residual=r)
        y = w(h, activation="swiglu")
        z = model.blocks[0].down(ops.quantize8(y), residual=s)
        tokens, logp = ops.sample(z, u, top_k=k, temperature=t, logprobs=True)
        return h.values(), z, tokens, logp
    ones = torch.ones(256, device=dev)
    k = torch.full((33,), 50, dtype=torch.int32, device=dev)
    t = torch.full((33,), 0.5, device=dev)
    inputs = [[torch.randn(33, 256, generator=g).to(dev), torch.randn(33, 256, generator=g).to(dev),
               torch.rand(33, generator=g).to(dev)] for _ in range(5)]
    want = [step(*i) for i in inputs]
    graphs = []
    for _ in range(2):
        held = [i.clone() for i in inputs[0]]
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(*held)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*held)
        graphs.append((graph, held, out))
    for i in range(5):
        for j, (graph, held, _) in enumerate(graphs):
            for a, b in zip(held, inputs[(i + j) % 5]):
                a.copy_(b)
            graph.replay()
        eager = step(*inputs[i])
        torch.cuda.synchronize()
        for j, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(i + j) % 5]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[i]))


def test_another_stream(dev, model):
    x = torch.randn(70, 256, device=dev)
    ones, u = torch.ones(256, device=dev), torch.rand(70, device=dev)
    w = model.blocks[1].attn.qkv

    def run(x):
        y = w(ops.rmsnorm8(x, ones))
        return y, ops.sample(y, u)
    want = run(x)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(x)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_what_a_model_in_8_bits_is_not_for(dev, model):
    with pytest.raises(ValueError, match="quantize_activations"):
        DecodeEngine(model)
    with pytest.raises(ValueError, match="quantize_activations"):
        to_nbpack_params(model)


def test_layers_that_do_not_fit_leave_the_model(dev):
    m = random_packed_model(ModelConfig(**CFG), seed=5, device=dev)
    down = m.blocks[1].ffn.down
    m.blocks[1].ffn.down = torch.nn.Linear(384, 256).to(dev)
    with pytest.raises(ValueError, match="3 bits"):
        quantize_activations(m)
    assert isinstance(m.blocks[0].attn.qkv, PackedLinear)
    with pytest.raises(ValueError, match="gate"):
        PackedLinear8.from_pairs(m.blocks[0].ffn.gate, down)


@pytest.mark.parametrize("N,K,activation", [(256, 384, None), (1000, 640, "gelu"), (2000, 256, "swiglu")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_do_not_depend_on_the_batch(dev, N, K, activation, dtype):
    g = torch.Generator().manual_seed(8)
    packed = ops.pack(torch.randint(0, 8, (N * K,), generator=g, dtype=torch.uint8).to(dev), 3)
    books = torch.randn(N * K // 128, 8, generator=g).to(dev)
    bias = torch.randn(N, generator=g).to(dev)
    layer = PackedLinear8.from_packed_linear(PackedLinear(packed, books, N, K), bias)
    x = torch.randn(2100, K, generator=g).to(dev, dtype)
    r = torch.randn(2100, N // 2 if activation == "swiglu" else N, generator=g).to(dev, dtype)
    weight = torch.rand(K, generator=g).to(dev)

    def run(rows):
        h = ops.rmsnorm8(x[rows], weight)
        return h, ops.quantize8(x[rows]), layer(h, activation=activation, residual=r[rows])
    h, q, y = run(slice(0, 2100))
    for rows in (slice(0, 1), slice(2090, 2099), slice(17, 57), slice(1, 130), slice(900, 1400)):
        h1, q1, y1 = run(rows)
        for a, b in ((h, h1), (q, q1)):
            assert torch.equal(a.codes[rows], b.codes) and torch.equal(a.scale[rows], b.scale)
        assert torch.equal(y[rows], y1)


def test_rows_far_apart(dev):
    """Inputs, sums, residuals and outputs whose rows pass 32 bits."""
    far, K, N = (1 << 30) + 16, 256, 48
    g = torch.Generator().manual_seed(16)

    def wide(t):
        out = torch.empty(2 * far + t.shape[1], dtype=t.dtype, device=dev).as_strided(t.shape, (far, 1))
        return out.copy_(t)
    x, y = (torch.randn(3, K, generator=g).to(dev) for _ in range(2))
    weight = torch.rand(K, generator=g).to(dev)
    packed = ops.pack(torch.randint(0, 8, (N * K,), generator=g, dtype=torch.uint8).to(dev), 3)
    w = ops.linear8_layout(packed, torch.randn(N * K // 128, 8, generator=g).to(dev), N, K)
    h, s = ops.rmsnorm8(x, weight, residual=y)
    a = wide(x)
    h1, s1 = ops.rmsnorm8(a, weight, residual=y, out=a)
    assert s1 is a and torch.equal(s, a) and torch.equal(h.codes, h1.codes) and torch.equal(h.scale, h1.scale)
    q, q1 = ops.quantize8(s), ops.quantize8(a)
    assert torch.equal(q.codes, q1.codes) and torch.equal(q.scale, q1.scale)
    r = torch.randn(3, N, generator=g).to(dev)
    out = wide(r)
    assert ops.linear8(q, w, residual=out, out=out) is out
    assert torch.equal(out, ops.linear8(q, w, residual=r))
