"""Drawn tokens on the GPU against extended precision on the host: the tokens
themselves, their log-probabilities within their rounding."""
import math

import numpy as np
import pytest
import torch

from nativebit_amd import ops
from tests import rows8_ref as ref

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def check(dev, logits, u, pad=0, **rules):
    """Every row against the reference; rules are lists or None."""
    B, V = logits.shape
    x = logits.to(dev)
    if pad:
        wide = torch.full((B, V + pad), 1e9, dtype=logits.dtype, device=dev)
        wide[:, 1:V + 1] = x
        x = wide[:, 1:V + 1]
    types = {"top_k": torch.int32}
    args = {k: torch.tensor(v, dtype=types.get(k, torch.float32)).to(dev) for k, v in rules.items()}
    ud = torch.tensor(u, dtype=torch.float32)
    tokens, logp = ops.sample(x, ud.to(dev), logprobs=True, **args)
    again = ops.sample(x, ud.to(dev), **args)
    assert torch.equal(tokens, again)
    for b in range(B):
        at = {k: v[b].item() for k, v in ((k, t.cpu()) for k, t in args.items())}
        token, lp = ref.sample(logits[b], ud[b].item(), **at)
        assert tokens[b].item() == token, (b, at, u[b])
        got = logp[b].item()
        # one rounding of a difference of two 64-bit logarithms
        assert got == lp or abs(got - lp) <= 2.0 ** -24 * abs(lp) + 1e-9, (b, got, lp)
    return tokens


def numbers(n, seed, low=0.0, high=1.0):
    return np.random.default_rng(seed).uniform(low, high, n).tolist()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 1023, 1025, 4097, 16385, 50257])
def test_sizes(dev, V, dtype):
    B = 6
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(B, V, generator=g) * 4).to(DT[dtype])
    for pad in (0, 3):
        check(dev, x, numbers(B, 1), pad)
        check(dev, x, numbers(B, 2), pad, temperature=numbers(B, 3, 0.2, 2))
    check(dev, x, numbers(B, 4), top_k=[1, 2, 5, 100, V, V + 1])
    check(dev, x, numbers(B, 5), top_p=[0.01, 0.3, 0.7, 0.9, 0.99, 1.0])
    check(dev, x, numbers(B, 6), min_p=[0.0, 0.001, 0.05, 0.5, 1.0, 2.0])
    check(dev, x, numbers(B, 7), temperature=numbers(B, 8, 0.5, 1.5), top_k=[0, 3, 50, 400, 2, 700],
          top_p=numbers(B, 9, 0.4, 1), min_p=numbers(B, 10, 0, 0.1))


@pytest.mark.parametrize("T", [0.3, 1.0, 5.0])
def test_many_draws(dev, T):
    """One row many times over: every border of the running sums is near some u."""
    V, B = 3000, 256
    row = torch.randn(V, generator=torch.Generator().manual_seed(3)) * 3
    x = row.expand(B, V).contiguous()
    u = ((torch.arange(B) + 0.5) / B).tolist()
    check(dev, x, u, temperature=[T] * B)
    check(dev, x, u, temperature=[T] * B, top_k=[500] * B, top_p=[0.9] * B)


def test_ties(dev):
    """Many equal logits: the lower tokens come first, and a cut runs through
    them."""
    B, V = 12, 5000
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-3, 4, (B, V), generator=g).float()
    for seed in range(3):
        u = numbers(B, seed)
        check(dev, x, u, top_k=[1, 2, 10, 700, 715, 720, 1400, 1500, 3000, 4999, 5000, 0])
        check(dev, x, u, top_p=numbers(B, seed + 10, 0.05, 0.95))
        check(dev, x, u, top_k=[900] * B, top_p=numbers(B, seed + 20, 0.3, 1), min_p=[0.1] * B)
    flat = torch.full((B, V), -2.5)
    check(dev, flat, numbers(B, 7), top_k=[0, 1, 2, 17, 63, 64, 65, 1000, 1024, 2500, 4999, 5000])
    check(dev, flat, numbers(B, 8), top_p=numbers(B, 9, 0.001, 0.999))


def test_numbers_at_the_ends(dev):
    x = torch.randn(4, 900, generator=torch.Generator().manual_seed(1))
    for u in (0.0, 1 - 2.0 ** -24, 1.0, -0.5, float("nan"), 1e-30):
        check(dev, x, [u] * 4)
        check(dev, x, [u] * 4, top_k=[1, 5, 40, 0], top_p=[0.9] * 4)


def test_masked_rows(dev):
    inf, nan = math.inf, math.nan
    x = torch.randn(9, 2100, generator=torch.Generator().manual_seed(2))
    x[0] = -inf                     # nothing is left
    x[1] = nan
    x[2, 5:] = -inf
    x[3, :2099] = -inf              # one token
    x[4, 100:200] = nan             # a NaN is never drawn
    x[5, [7, 70, 700]] = inf        # only they are
    x[6, 9] = inf
    x[7, ::2] = -inf
    x[8] = -3.4e38
    x[8, 1] = 3.4e38
    for rules in ({}, {"top_k": [2] * 9}, {"top_p": [0.5] * 9}, {"min_p": [0.2] * 9},
                  {"temperature": [0.7] * 9, "top_k": [40] * 9, "top_p": [0.8] * 9, "min_p": [0.01] * 9}):
        for seed in range(3):
            t = check(dev, x, numbers(9, seed), **rules)
            assert t[0] == -1 and t[1] == -1 and t[3] == 2099 and t[6] == 9
            assert t[5].item() in (7, 70, 700) and t[2] < 5


def test_temperatures(dev):
    inf, nan = math.inf, math.nan
    T = [0.0, -1.0, nan, 1e-30, 1e-45, 1e-4, 100.0, 1e30, inf]
    x = torch.randn(len(T), 3000, generator=torch.Generator().manual_seed(4))
    x[:, 1000:1500] = -inf
    x[:, 2000] = x[:, 2500] = 9.0   # the largest twice
    for seed in range(3):
        t = check(dev, x, numbers(len(T), seed), temperature=T)
        assert (t[:3] == 2000).all()
        check(dev, x, numbers(len(T), seed), temperature=T, top_k=[30] * len(T), top_p=[0.6] * len(T))


def test_rules_that_keep_all_or_one(dev):
    x = torch.randn(8, 1500, generator=torch.Generator().manual_seed(6))
    u = numbers(8, 1)
    plain = check(dev, x, u)
    nan = math.nan
    for rules in ({"top_k": [0, -1, 1500, 2000] * 2}, {"top_p": [1.0, 2.0, nan, math.inf] * 2},
                  {"min_p": [0.0, -1.0, nan, 0.0] * 2}):
        assert torch.equal(check(dev, x, u, **{k: [nan if z != z else z for z in v]
                                               for k, v in rules.items()}), plain)
    best = x.argmax(1)
    for rules in ({"top_k": [1] * 8}, {"top_p": [0.0, -1.0, 1e-30, 1e-9] * 2}, {"min_p": [1.0, 2.0] * 4}):
        assert torch.equal(check(dev, x, u, **rules).long().cpu(), best)


def test_large_vocabulary(dev):
    B, V = 3, 131077
    x = torch.randn(B, V, generator=torch.Generator().manual_seed(8)) * 4
    check(dev, x, numbers(B, 1), temperature=[0.8, 1.0, 1.3], top_k=[0, 1000, 50], top_p=[0.95, 0.9, 1.0],
          min_p=[0.0, 0.0, 0.05])
    check(dev, x.to(torch.bfloat16), numbers(B, 2), top_p=[0.95, 0.6, 0.999])


def test_no_rows(dev):
    tokens, logp = ops.sample(torch.empty(0, 10, device=dev), torch.empty(0, device=dev), logprobs=True)
    assert tokens.shape == (0,) and logp.shape == (0,)


KS = [1, 2, 63, 64, 65, 200, 626, 627, 1000, 1024, 1500, 3000]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("order", ["rising", "falling", "blocks", "any"])
def test_few_or_many_kept(dev, dtype, order):
    """Tokens that top_k keeps next to each other, more of them among 64
    neighbours than can be listed, many that are equal."""
    B, V = len(KS), 20011
    x = torch.randn(B, V, generator=torch.Generator().manual_seed(11)) * 2
    if order == "rising":
        x = x.sort(1).values
    elif order == "falling":
        x = x.sort(1, descending=True).values
    elif order == "blocks":
        x = x[:, :V // 64 + 1].repeat_interleave(64, 1)[:, :V].contiguous()
    x = x.to(DT[dtype])
    u = numbers(B, 1)
    check(dev, x, u, top_k=KS)
    check(dev, x, u, pad=5, top_k=KS[::-1], top_p=numbers(B, 2, 0.2, 1), temperature=numbers(B, 3, 0.3, 30))
    check(dev, x, u, top_k=[2000] * B, top_p=numbers(B, 4, 0.2, 1), min_p=numbers(B, 5, 0, 0.01))
    x[:, 100:19000] = -math.inf
    check(dev, x, u, top_k=KS)
    x[:, 5:] = -math.inf
    check(dev, x, u, top_k=KS, temperature=numbers(B, 6, 0.3, 30))


def test_more_equal_groups_than_are_looked_into(dev):
    V = 300001
    x = torch.zeros(3, V)
    x[1, ::3] = 1.0
    x[2, 299_000] = 2.0
    check(dev, x, [0.1, 0.5, 0.99], top_k=[500, 1000, 1024])
    check(dev, x, [0.1, 0.5, 0.99], top_k=[500, 1000, 1024], top_p=[0.7] * 3)


def test_most_of_a_large_vocabulary_kept(dev):
    """top_k around the largest that is looked up in groups."""
    ks = [1023, 1024, 1025, 2047, 2048, 2049]
    x = torch.randn(6, 100003, generator=torch.Generator().manual_seed(12)) * 3
    check(dev, x, numbers(6, 1), top_k=ks, temperature=[5.0] * 6)
    check(dev, x, numbers(6, 2), top_k=ks, top_p=[0.97] * 6, min_p=[1e-3] * 6)


def test_vocabularies_of_many_groups(dev):
    """More groups of 32 tokens than are looked at together."""
    B, V = 4, 300001
    x = torch.randn(B, V, generator=torch.Generator().manual_seed(13)) * 3
    check(dev, x, numbers(B, 1), top_k=[3, 100, 2048, 2049])
    check(dev, x, numbers(B, 2), top_p=[0.3, 0.9, 0.99, 0.9999], temperature=[1.0, 1.0, 1.5, 3.0])
    check(dev, x, numbers(B, 3), min_p=[0.5, 1e-2, 1e-4, 1e-6])


@pytest.mark.parametrize("rules", [{}, {"top_k": 700}, {"top_k": 2900}, {"top_p": 0.97}, {"min_p": 1e-3},
                                   {"top_k": 200, "top_p": 0.8, "min_p": 1e-3}])
def test_largest_vocabulary(dev, rules):
    """2^24 tokens, all but 3000 of them masked, against those 3000 by themselves (their
    weights are whole numbers of 2^-38 and 2^-45: u is not near a border)."""
    B, V, n = 3, 1 << 24, 3000
    g = torch.Generator().manual_seed(14)
    few = (torch.randn(B, n, generator=g) * 3).to(dev)
    at = torch.randperm(V, generator=g)[:n].sort().values.to(dev)
    x = torch.full((B, V), -math.inf, device=dev)
    x[:, at] = few
    args = {k: torch.full((B,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device=dev)
            for k, v in rules.items()}
    for u in ([0.1, 0.5, 0.9], [0.3141, 0.001, 0.77]):
        u = torch.tensor(u, device=dev)
        want, lp = ops.sample(few, u, logprobs=True, **args)
        got, lq = ops.sample(x, u, logprobs=True, **args)
        assert torch.equal(at[want.long()].int(), got)
        # (sums of up to 3000 weights that are half of 2^-38 off, of 1 or more; fp32's half step)
        assert ((lp - lq).abs() <= 3000 * 2.0 ** -38 + 2.0 ** -24 * lp.abs() * 2).all()


def test_rows_far_apart(dev):
    """Rows whose elements' numbers and bytes pass 32 bits."""
    far, V = (1 << 31) + 24, 700
    x = torch.randn(3, V, generator=torch.Generator().manual_seed(15)).to(torch.bfloat16)
    wide = torch.empty(2 * far + V, dtype=torch.bfloat16, device=dev).as_strided((3, V), (far, 1))
    wide.copy_(x)
    u = torch.tensor([0.2, 0.6, 0.95], device=dev)
    for k in (None, torch.tensor([5, 40, 0], dtype=torch.int32, device=dev)):
        assert torch.equal(ops.sample(wide, u, top_k=k), ops.sample(x.to(dev), u, top_k=k))
