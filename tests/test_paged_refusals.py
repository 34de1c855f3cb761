"""PagedCache and generate without a GPU: what they refuse on the host."""
import types

import pytest
import torch

from nativebit_amd import paged


def shape(**kw):
    a = dict(n_head=4, n_embd=256, context_len=300, n_layers=2)
    return types.SimpleNamespace(**{**a, **kw})


@pytest.mark.parametrize("kw", [dict(n_blocks=0), dict(max_requests=0), dict(max_len=0), dict(max_len=301)])
def test_cache_sizes(kw):
    with pytest.raises(ValueError):
        paged.PagedCache(shape(), **{"n_blocks": 4, "max_requests": 2, "device": "cpu", **kw})


@pytest.mark.parametrize("C,H", [(256, 32), (264, 3), (1024, 2)])
def test_cache_head_dims(C, H):
    with pytest.raises(ValueError):
        paged.PagedCache(shape(n_embd=C, n_head=H), 4, 2, device="cpu")


def test_steps_are_checked_on_the_host():
    c = paged.PagedCache(shape(), 4, 2, device="cpu")
    assert len(c) == 2 and c.table.shape == (2, 5) and (c.table == -1).all()
    for new in ([1, 1, 1], [-1, 2], [301, 0], [0, 257], [129, 65]):
        with pytest.raises(ValueError):
            c.step(new)
    with pytest.raises(ValueError):
        c.step([1, 1], n_tokens=3)
    with pytest.raises(ValueError):
        c.step(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        c.step([1, 1], prefix=[3])
    for _ in range(2):                   # fits, but there is no CPU implementation: nothing changes
        with pytest.raises(ValueError):
            c.step([128, 65])
    with pytest.raises(ValueError):
        c.release([2])
    with pytest.raises(IndexError):
        c[2]
    with pytest.raises(ValueError):      # no step planned
        c[0].attend(torch.zeros(1, 768), None, None, 4)


def test_generate_refuses():
    model = types.SimpleNamespace(embedding=types.SimpleNamespace(weight=torch.zeros(10, 4)),
                                  context_len=20)
    for n in (20, 100):
        with pytest.raises(ValueError):
            paged.generate(model, [[1], [2, 3]], n)
    for prompts in ([], [[]], [[1], []], [[10]], [[-1]]):
        with pytest.raises(ValueError):
            paged.generate(model, prompts, 1)
    with pytest.raises(ValueError, match="bias"):
        paged.generate(model, [[1], [2, 3]], 1, bias=[{1: 2.0}])
    cache = paged.PagedCache(shape(context_len=20), 4, 2, device="cpu")
    cache.lens[1] = 3
    with pytest.raises(ValueError, match="holds requests"):
        paged.generate(model, [[1], [2, 3]], 1, cache=cache)
