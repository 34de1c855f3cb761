"""paged.generate's top_k without a GPU: whole numbers of any width, one or one for
each request, reach the draw as int32 that keep what they say."""
import types

import numpy as np
import pytest
import torch

from nativebit_amd import ops, paged


class Cache:
    max_len, lens, table, state = 20, torch.zeros(2), torch.zeros(2, 1), torch.tensor([9])

    def step(self, lengths):
        pass


@pytest.fixture
def drawn(monkeypatch):
    """generate of one token for two prompts; the rules that ops.sample gets."""
    got = {}

    def sample(logits, u, **rules):
        got.update(rules)
        return torch.zeros(2, dtype=torch.int32)
    monkeypatch.setattr(ops, "sample", sample)
    monkeypatch.setattr(ops, "logits_rules", lambda logits, out, **rules: out)
    model = types.SimpleNamespace(embedding=types.SimpleNamespace(weight=torch.zeros(10, 4)), context_len=20,
                                  hidden=lambda idx, cache: (torch.zeros(1, 3, 4), cache),
                                  head=lambda h: torch.zeros(2, 10))

    def run(top_k):
        paged.generate(model, [[1], [2, 3]], 1, temperature=1.0, top_k=top_k, cache=Cache())
        return got["top_k"]
    return run


MOST = 2 ** 31 - 1


@pytest.mark.parametrize("top_k,want", [
    (3, [3, 3]), ([4, 0], [4, 0]), (MOST, [MOST] * 2), (1 << 31, [MOST] * 2), ((1 << 32) + 5, [MOST] * 2),
    ([1, 1 << 40], [1, MOST]), (torch.tensor([(1 << 32) + 5, 7]), [MOST, 7]),
    (np.array([7, (1 << 33) + 1]), [7, MOST]), (torch.tensor([200, 3], dtype=torch.uint8), [200, 3]),
    (-1, [0, 0]), ([-(1 << 40), 2], [0, 2]), (torch.tensor(9), [9, 9])])
def test_whole_numbers_of_any_width(drawn, top_k, want):
    got = drawn(top_k)
    assert got.dtype == torch.int32 and got.tolist() == want


@pytest.mark.parametrize("top_k", [2.0, [1, 2.5], torch.tensor([1.0, 2.0]), 1j, np.float64(3)])
def test_other_numbers_are_refused(drawn, top_k):
    with pytest.raises(ValueError, match="whole"):
        drawn(top_k)
