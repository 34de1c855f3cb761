"""PagedCache and generate on the GPU: a model's steps over requests that
come, grow and end, every layer's attention against 64 bits; batches against
requests one by one; rules on the choice."""
import numpy as np
import pytest
import torch

from nativebit_amd import ops, paged
from nativebit_amd.model import ModelConfig, random_packed_model
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(dev):
    cfg = ModelConfig(vocab_size=300, n_layers=2, n_embd=256, n_head=4, ffn_hidden=384, context_len=400)
    return random_packed_model(cfg, seed=5, device=dev)


def checked_attend(monkeypatch):
    """Every layer's attention checked against the definitions on what the
    cache holds (the bound of test_gpu_serving's attention)."""
    seen = []
    attend = paged.PagedLayer.attend

    def check(self, qkv, cos, sin, n_head):
        out = attend(self, qkv, cos, sin, n_head)
        c, i = self.cache, self.index
        plan = [t.cpu().numpy() for t in c.plan]
        slots, pos, chunks, lens = plan[:4]
        D = c.head_dim
        x = qkv.cpu().double().numpy()[:, :n_head * D].reshape(-1, n_head, D)
        t = [a.cpu().double().numpy()[pos][:, None] for a in (cos, sin)]
        q = (ref.rope(x, *t) / D ** 0.5).reshape(-1, n_head * D)
        cache = [a[i].cpu().numpy() for a in (c.k, c.v, c.k_scale, c.v_scale)]
        kw = {"softcap": c.softcap, "window": c.window}
        if c.slopes is not None:
            kw["slopes"] = c.slopes.cpu().numpy()
        if c.prefix is not None:
            kw["prefix"] = c.prefix.cpu().numpy()
        want, loss, top = ref.attention(q, chunks, c.table.cpu().numpy(), *cache, lens, **kw)
        u, blocks = 2.0 ** -24, 1 + int(lens.max()) // 64
        # (q is the kernel's fp32 one here: five roundings more, in the products' size)
        bound = ((2 * 16 * u * loss + 64 * u + (14 + 3 * blocks) * u) * top)[..., None]
        got = out.cpu().numpy().reshape(want.shape)
        ok = slots >= 0
        assert (np.abs(got - want)[ok] <= bound[ok]).all()
        assert (got[~ok] == 0).all()
        seen.append(i)
        return out
    monkeypatch.setattr(paged.PagedLayer, "attend", check)
    return seen


@pytest.mark.parametrize("rules", [{}, {"softcap": 4.0, "window": 40, "slopes": [0.5, 0.1, 0.02, 0.0]}])
def test_steps(dev, model, monkeypatch, rules):
    seen = checked_attend(monkeypatch)
    c = paged.PagedCache(model, 14, 4, **rules)
    g = torch.Generator().manual_seed(1)

    def step(new, **kw):
        before = len(seen)
        p = c.step(new, **kw)
        idx = torch.randint(0, 300, (1, p.slots.shape[0]), generator=g).to(dev)
        logits, back = model(idx, kv_caches=c)
        assert back is c and logits.shape == (1, idx.shape[1], 300)
        assert seen[before:] == [0, 1]
        return logits
    step([100, 1, 0, 65])
    step([1, 1, 0, 1], prefix=[50, 0, 9, 300])
    step([0, 190, 3, 0])
    assert c.lens.tolist() == [101, 192, 3, 66] and c.state.tolist() == [14 - 2 - 3 - 1 - 2, 0]
    c.release([1, 3])
    assert c.lens.tolist() == [101, 0, 3, 0] and c.state.tolist()[0] == 11
    with pytest.raises(ValueError):
        c.step([1, 400, 400, 1])
    step([28, 330, 1, 60])
    assert sorted(c.table[c.table >= 0].tolist()) == sorted(set(c.table[c.table >= 0].tolist()))
    # counts that only the GPU knows, rows behind the last request's
    new = torch.tensor([1, 1, 0, 7], dtype=torch.int32, device=dev)
    logits = step(new, n_tokens=12)
    assert torch.isfinite(logits).all()
    step([1, 1, 1, 1])
    assert c.lens.tolist() == [131, 332, 5, 68]
    keys, values = c.read(1, 2)
    assert keys.shape == values.shape == (4, 5, 64)


def test_blocks_run_out_on_the_gpu(dev, model):
    """From a tensor the step goes on: tokens without room have no slot."""
    c = paged.PagedCache(model, 3, 3)
    new = torch.tensor([100, 50, 70], dtype=torch.int32, device=dev)
    p = c.step(new, n_tokens=220)
    logits, _ = model(torch.ones(1, 220, dtype=torch.int64, device=dev), kv_caches=c)
    assert c.lens.tolist() == [100, 50, 0] and c.state.tolist() == [0, 70]
    assert (p.slots[150:] == -1).all() and torch.isfinite(logits).all()
    c.release([0])
    p = c.step([0, 10, 60])
    assert c.lens.tolist() == [0, 60, 60] and (p.slots >= 0).all()


def test_generate_is_each_request_alone(dev, model):
    """A batch's continuations are those of its requests alone (chosen tokens:
    the logits differ in the order of fp32 sums)."""
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (70, 1, 129, 20, 64)]
    together = paged.generate(model, prompts, 20)
    alone = [paged.generate(model, [p], 20)[0] for p in prompts]
    assert together == alone
    assert all(len(t) == 20 and 0 <= min(t) and max(t) < 300 for t in together)
    assert paged.generate(model, prompts, 0) == [[]] * 5


def test_generate_rules(dev, model):
    prompts = [[3, 5, 3], [7], [9, 9, 9, 9]]
    # a penalty for each time: no token comes twice before all have
    out = paged.generate(model, prompts, 100, frequency=1000.0)
    assert all(len(set(o)) == 100 for o in out)
    # only even tokens; one request has none
    mask = torch.full((3, 10), 0x55555555, dtype=torch.int32, device=dev)
    mask[1] = 0
    out = paged.generate(model, prompts, 8, mask=mask)
    assert all(t % 2 == 0 for o in (out[0], out[2]) for t in o) and out[1] == [-1] * 8
    # biases: one token forced, one request's first choice banned, one free
    free = paged.generate(model, prompts, 4)
    out = paged.generate(model, prompts, 4, bias=[{11: 1e4}, {free[1][0]: -1e4}, {}])
    assert out[0] == [11] * 4 and free[1][0] not in out[1] and out[2] == free[2]
    # a repetition penalty: the choice of the plain restatement, step by step
    cache = paged.PagedCache(model, 8, 3)
    out = paged.generate(model, prompts, 6, repetition=[1.5, 1.0, 3.0], presence=0.3, cache=cache)
    assert cache.lens.tolist() == [3 + 5, 1 + 5, 4 + 5]
    seq = [list(p) for p in prompts]
    cache = paged.PagedCache(model, 8, 3)
    feed = prompts
    for i in range(6):
        cache.step([len(f) for f in feed])
        logits, _ = model(torch.tensor([sum(feed, [])], device=dev), kv_caches=cache)
        rows = np.cumsum([len(f) for f in feed]) - 1
        hist = np.full((3, 20), -1)
        for r, s in enumerate(seq):
            hist[r, :len(s)] = s
        _, tokens = ref.rules(logits[0, rows].cpu().numpy(), hist, [len(s) for s in seq],
                              [len(p) for p in prompts], [1.5, 1.0, 3.0], None, [0.3] * 3)
        assert tokens.tolist() == [o[i] for o in out]
        feed = [[int(t)] for t in tokens]
        for s, f in zip(seq, feed):
            s += f


def test_decode_step_in_a_graph(dev, model):
    """A whole decode step of a batch -- plan, layers, head, rules -- captured
    once and replayed, against the same steps run eagerly."""
    prompts = [[5, 6, 7] * 20, [1], [2] * 63]
    eager = paged.generate(model, prompts, 12, repetition=1.2)
    c = paged.PagedCache(model, 20, 3)
    width = 80
    history = torch.full((3, width), -1, dtype=torch.int32, device=dev)
    for r, p in enumerate(prompts):
        history[r, :len(p)] = torch.tensor(p, dtype=torch.int32)
    lens = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=dev)
    rep = torch.full((3,), 1.2, device=dev)
    c.step([len(p) for p in prompts])
    with torch.no_grad():
        hidden, _ = model.hidden(torch.tensor([sum(prompts, [])], device=dev), c)
        logits = model.head(hidden[0, lens.long().cumsum(0) - 1])
    _, tok = ops.logits_rules(logits, history=history, lens=lens, repetition=rep, choose=True)
    tokens, ones = tok.clone(), torch.ones(3, dtype=torch.int32, device=dev)
    state = [t.clone() for t in (c.table, c.lens, c.state, history, lens, tokens, c.k, c.v,
                                 c.k_scale, c.v_scale)]

    def one():
        history.scatter_(1, lens.long()[:, None], tokens[:, None])
        lens.add_(1)
        c.step(ones, n_tokens=3)
        with torch.no_grad():
            hidden, _ = model.hidden(tokens.long()[None], c)
            logits = model.head(hidden[0])
        tokens.copy_(ops.logits_rules(logits, history=history, lens=lens, repetition=rep, choose=True)[1])
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        one()
    torch.cuda.current_stream().wait_stream(s)
    for t, b in zip((c.table, c.lens, c.state, history, lens, tokens, c.k, c.v, c.k_scale, c.v_scale), state):
        t.copy_(b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        one()
    out = [tokens.tolist()]
    for _ in range(11):
        g.replay()
        out.append(tokens.tolist())
    assert [list(o) for o in zip(*out)] == eager
