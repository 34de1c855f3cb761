"""Slopes and prefixes of a PagedCache: slope * (key's position - query's) is a
penalty by distance up to the query only, so a token that sees others behind it,
inside a prefix, is refused."""
import pytest
import torch

from nativebit_amd import paged
from tests.test_paged_refusals import shape


def stepped(new, prefix, slopes, known=(0, 0)):
    c = paged.PagedCache(shape(), 10, 2, slopes=slopes, device="cpu")
    c._known, c._left = list(known), 10 - sum(-(-k // 64) for k in known)
    c.step(new, n_tokens=2 if isinstance(new, torch.Tensor) else None, prefix=prefix)


SLOPES = [0.5, 0.1, 0.0, 0.2]


@pytest.mark.parametrize("new,prefix,known", [
    ([20, 0], [2, 0], (0, 0)), ([20, 1], [20, 0], (0, 0)), ([1, 2], [0, 300], (0, 90)),
    ([5, 5], torch.tensor([0, 12]), (20, 10)),
    (torch.ones(2, dtype=torch.int32), [0, 1], (0, 0)),
])
def test_tokens_inside_a_prefix(new, prefix, known):
    with pytest.raises(ValueError, match="slopes"):
        stepped(new, prefix, SLOPES, known)
    with pytest.raises(ValueError, match="GPU"):      # without them the plan is next
        stepped(new, prefix, None, known)


@pytest.mark.parametrize("new,prefix,known", [
    ([20, 3], [1, 0], (0, 0)),                  # a prefix of the first token
    ([1, 1], [50, 300], (100, 65)),             # single tokens see none behind them
    ([5, 0], [20, 9], (20, 4)),                 # behind the prefix; no tokens
    ([5, 5], [21, 11], (20, 10)),
])
def test_tokens_behind_a_prefix(new, prefix, known):
    with pytest.raises(ValueError, match="GPU"):
        stepped(new, prefix, SLOPES, known)
