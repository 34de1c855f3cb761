"""generate in a cache of the caller's: without room for all of it nothing is
begun."""
import types

import pytest
import torch

from nativebit_amd import paged


def cache(n_blocks, max_requests):
    shape = types.SimpleNamespace(n_head=4, n_embd=256, context_len=300, n_layers=2)
    return paged.PagedCache(shape, n_blocks, max_requests, device="cpu")


class Model:
    context_len = 300
    embedding = types.SimpleNamespace(weight=torch.zeros(10, 4))

    def hidden(self, idx, kv_caches):
        raise AssertionError("begun")


@pytest.mark.parametrize("blocks,requests,lengths,n,fits", [
    (4, 2, (1, 2, 3), 1, False),            # requests
    (2, 3, (1, 2, 3), 1, False), (3, 3, (1, 2, 3), 1, True),
    (3, 2, (60, 64), 5, True),              # 64 and 68 tokens at the end
    (3, 2, (60, 64), 6, False), (4, 2, (60, 64), 6, True),
    (4, 1, (200,), 57, True), (4, 1, (200,), 58, False),
])
def test_generate_asks_for_room_first(blocks, requests, lengths, n, fits):
    c = cache(blocks, requests)
    # (with room the plan is next, for which there is no CPU implementation)
    with pytest.raises(ValueError, match="GPU|cuda|device" if fits else "requests of"):
        paged.generate(Model(), [[1] * k for k in lengths], n, cache=c)
    assert c.plan is None and c.state.tolist() == [blocks, 0]
    assert paged.generate(Model(), [[1] * k for k in lengths], 0, cache=c) == [[] for _ in lengths]
