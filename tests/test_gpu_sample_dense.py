"""Drawn tokens of dense rows of millions of tokens on the GPU: slices longer than 2^14,
sums near 2^62, rows whose cuts are looked for in the whole row.  Their tokens follow in
closed form: rows of a few values, whose order is by value and then by token."""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from nativebit_amd import ops

pytestmark = pytest.mark.gpu


def draw(dev, row, us, dtype=torch.float32, **rules):
    """(tokens, logprobs) of one row of logits for several numbers."""
    n = len(us)
    x = row.to(dev, dtype).expand(n, -1).contiguous()
    args = {k: torch.full((n,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device=dev)
            for k, v in rules.items()}
    tokens, logp = ops.sample(x, torch.tensor(us, device=dev), logprobs=True, **args)
    return tokens.tolist(), logp.tolist()


def kept_of_flat(V, rules):
    """How many tokens of a flat row are kept: whole weights, shares of them."""
    k = min(rules.get("top_k", V), V)
    if "top_p" in rules:
        k = max(math.ceil(Fraction(float(np.float32(rules["top_p"]))) * k), 1)
    return k


US = [0.0, 0.1, 0.4999, 0.5, 0.77, 0.999999]


@pytest.mark.parametrize("V", [(1 << 21) + 3, 1 << 22, (1 << 24) - 1, 1 << 24])
@pytest.mark.parametrize("rules", [{}, {"top_p": 0.75}, {"top_k": 2048}, {"top_k": 2049}, {"top_k": 1500001},
                                   {"top_k": 1500001, "top_p": 0.3}, {"min_p": 0.5}])
def test_flat_rows(dev, V, rules):
    """Every weight is 1: the first of the order are the first tokens, the token of u is
    floor(u n) of n kept ones."""
    n = kept_of_flat(V, rules)
    # (top_p's share is rounded up to a whole multiple of 2^-38 or finer: the same number
    # of whole weights)
    us = [float(np.float32(u)) for u in US]
    tokens, logp = draw(dev, torch.full((V,), -3.25), us, **rules)
    assert tokens == [int(Fraction(u) * n) for u in us]
    assert all(abs(lp + math.log(n)) <= 2.0 ** -23 * math.log(n) + 1e-9 for lp in logp)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rules", [{}, {"top_p": 0.6}, {"top_k": 3000000}, {"top_k": 2000000, "top_p": 0.9, "min_p": 0.3},
                                   {"min_p": 0.2}, {"min_p": 0.05}])
def test_rows_of_three_values(dev, rules, dtype):
    """Logits 0, -1 and -2.5 in turn by token, over 2^22 tokens.  u is taken in the middle
    of a token's weight, where no rounding of weights (2^-40 each) moves it."""
    V = (1 << 22) + 5
    values = [-1.0, 0.0, -2.5]
    row = torch.tensor(values).repeat(V // 3 + 1)[:V]
    ids = np.arange(V)
    value = np.array(values)[ids % 3]
    order = np.argsort(-value, kind="stable")
    w = np.exp(value)
    kept = order[:rules.get("top_k", V)]
    if "top_p" in rules:
        upto = np.cumsum(w[kept].astype(np.longdouble))
        total = upto[-1]
        share = np.longdouble(np.float32(rules["top_p"])) * total
        n = int(np.searchsorted(upto, share, side="left")) + 1
        # (the cut is not within a rounding of a border)
        assert min(abs(upto[n - 1] - share), abs(share - upto[n - 2])) > 1e-4
        kept = kept[:n]
    if "min_p" in rules:
        kept = kept[w[kept] >= rules["min_p"]]
    kept = np.sort(kept)
    upto = np.cumsum(w[kept].astype(np.longdouble))
    total = upto[-1]
    picks = [0, 1, 1000, len(kept) // 3, len(kept) // 2 + 1, len(kept) - 1]
    us, want = [], []
    for i in picks:
        u = min(np.float32((upto[i] - w[kept[i]] / 2) / total), np.float32(1 - 2.0 ** -24))
        j = int(np.searchsorted(upto, np.longdouble(u) * total, side="right"))     # (u as fp32 holds it)
        near = np.longdouble(u) * total
        if min(abs(upto[j] - near), abs(near - (upto[j] - w[kept[j]]))) > 1e-4:
            us.append(float(u)), want.append(int(kept[j]))
    assert len(us) >= 4
    tokens, logp = draw(dev, row, us, dtype, **rules)
    assert tokens == want
    for t, lp in zip(tokens, logp):
        exact = value[t] - float(np.log(total))
        # (V weights half of 2^-40 off each, relative to the total; one rounding)
        assert abs(lp - exact) <= 2.0 ** -24 * abs(exact) + V * 2.0 ** -41 / float(total) + 1e-9
