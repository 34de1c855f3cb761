"""Requests that may not fill their tables (a context that is no multiple of 64
tokens): the plan against a restatement token by token, and a PagedCache of such
a model from lists and from counts on the GPU."""
import numpy as np
import pytest
import torch

from nativebit_amd import ops, paged
from nativebit_amd.model import ModelConfig, random_packed_model
from tests import serving_ref as ref
from tests.test_gpu_serving import dev_i32, host

pytestmark = pytest.mark.gpu


def restated(table, lens, new, free, state, n_tokens, most):
    """(table, slots, positions, chunks, lens, state): every token of every
    request in order takes a row, and a slot while its request may grow."""
    table, free = table.copy(), list(free[:int(state[0])])
    slots, positions = np.full(n_tokens, -1), np.zeros(n_tokens, dtype=np.int64)
    ends, runs, row, dropped = lens.copy(), [], 0, 0
    for r in range(len(lens)):
        full = False
        for p in range(lens[r], lens[r] + new[r]):
            row += 1
            full = full or p >= min(most, table.shape[1] * 64) or (p % 64 == 0 and not free)
            if full or row > n_tokens:
                dropped += 1
                continue
            if p % 64 == 0:
                table[r, p // 64] = free.pop()
            slots[row - 1], positions[row - 1], ends[r] = 64 * table[r, p // 64] + p % 64, p, p + 1
            if runs and runs[-1][2] == r and runs[-1][3] // 64 == p // 64:
                runs[-1][1] += 1
            else:
                runs.append([row - 1, 1, r, p])
    chunks = np.zeros((ops.kv_plan_chunks(n_tokens, len(lens)), 4), dtype=np.int64)
    chunks[:len(runs)] = np.array(runs).reshape(-1, 4)
    return table, slots, positions, chunks, ends, np.array([len(free), dropped])


@pytest.mark.parametrize("most", [1, 63, 64, 65, 100, 200, 255, 256, 300, 1 << 40])
@pytest.mark.parametrize("R,n_new,spare", [(1, 150, 9), (5, 90, 20), (300, 40, 250), (300, 7, 3)])
def test_plan_max_len(dev, most, R, n_new, spare):
    rng = np.random.default_rng(R + spare)
    lens = rng.integers(0, min(most, 256) + 1, R)
    new = rng.integers(0, n_new + 1, R)
    table, free, state = ref.tables(lens, 4, int((-(-lens // 64)).sum()) + spare, rng)
    for rows in (int(new.sum()), int(new.sum()) // 2, int(new.sum()) + 5):
        want = restated(table, lens, new, free, state, rows, most)
        t = dev_i32(table, dev)
        p = ops.kv_plan(t, *(dev_i32(a, dev) for a in (lens, new, free, state)), rows, max_len=most)
        for name, a, b in zip(("table", "slots", "positions", "chunks", "lens", "state"), (t, *p), want):
            assert np.array_equal(host(a), b), name


def test_plan_of_requests_that_are_too_long(dev):
    """A request that has more than it may have keeps its tokens and gets none."""
    lens = np.array([130, 60, 100])
    table, free, state = ref.tables(lens, 4, 20, np.random.default_rng(0))
    t = dev_i32(table, dev)
    p = ops.kv_plan(t, *(dev_i32(a, dev) for a in (lens, [5, 45, 3], free, state)), 53, max_len=100)
    # (three, one and two of 20 blocks held, one more taken; 5 + 5 + 3 tokens left out)
    assert host(p.lens).tolist() == [130, 100, 100] and host(p.state).tolist() == [20 - 6 - 1, 13]
    assert (host(p.slots) >= 0).tolist() == [False] * 5 + [True] * 40 + [False] * 8


@pytest.mark.parametrize("max_len", [None, 70])
def test_cache_keeps_its_length(dev, max_len):
    cfg = ModelConfig(vocab_size=300, n_layers=2, n_embd=128, n_head=2, ffn_hidden=128, context_len=100)
    model = random_packed_model(cfg, seed=3, device=dev)
    c = paged.PagedCache(model, 6, 3, max_len)
    most = max_len or 100
    assert c.max_len == most

    def step(new, n):
        p = c.step(dev_i32(new, dev), n_tokens=n)
        logits, _ = model(torch.ones(1, n, dtype=torch.int64, device=dev), kv_caches=c)
        return p, logits
    p, logits = step([most - 2, 1, 200], most + 199)
    assert c.lens.tolist() == [most - 2, 1, most] and c.state.tolist() == [6 - 5, 200 - most]
    slots = host(p.slots)
    assert (slots[:most - 1] >= 0).all() and (slots[most - 1:2 * most - 1] >= 0).all()
    assert (slots[2 * most - 1:] == -1).all() and torch.isfinite(logits).all()
    for i in range(4):
        p, logits = step([1, 1, 1], 3)
        assert host(p.slots >= 0).tolist() == [i < 2, True, False] and torch.isfinite(logits).all()
        assert c.state[1] == (1 if i < 2 else 2)
    assert c.lens.tolist() == [most, 5, most]
    for layer in range(2):
        for r in range(3):
            for t in c.read(layer, r):
                assert torch.isfinite(t).all() and t.abs().sum() > 0
    # from a list again: refused past the length, right up to it
    with pytest.raises(ValueError, match="max_len"):
        c.step([1, 0, 0])
    c.step([0, most - 5, 0])
    with pytest.raises(ValueError, match="max_len"):
        c.step([0, 1])
    assert c.lens.tolist() == [most] * 3
