"""The serving operators on the GPU against their plain restatements: the plan
and the codes bit for bit, attention within a bound derived from its
roundings, rules on logits bit for bit."""
import math

import numpy as np
import pytest
import torch

from nativebit_amd import ops
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def dev_i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(dev)


def host(t):
    return t.cpu().numpy()


# ---------------------------------------------------------------------------
# plan and release
# ---------------------------------------------------------------------------
def run_plan(dev, table, lens, new, free, state, n, stride=None):
    t = dev_i32(table, dev)
    if stride:
        wide = torch.full((table.shape[0], stride), 77, dtype=torch.int32, device=dev)
        wide[:, :table.shape[1]] = t
        t = wide[:, :table.shape[1]]
    args = [dev_i32(a, dev) for a in (lens, new, free, state)]
    before = [a.clone() for a in args]
    p = ops.kv_plan(t, *args, n)
    again = ops.kv_plan(t, *args, n)
    for a, b in zip(args, before):
        assert torch.equal(a, b)
    for a, b in zip(p, again):
        assert torch.equal(a, b)
    if stride:
        assert (wide[:, table.shape[1]:] == 77).all()
    return t, p


def check_plan(dev, table, lens, new, free, state, n, stride=None):
    want = ref.plan(table, lens, new, free, state, n)
    t, p = run_plan(dev, table, lens, new, free, state, n, stride)
    for name, a, b in zip(("table", "slots", "positions", "chunks", "lens", "state"), (t, *p), want):
        assert np.array_equal(host(a), b), name
    return t, p


@pytest.mark.parametrize("R,width,longest,n_new,spare,seed", [
    (1, 1, 0, 1, 0, 0), (1, 1, 63, 1, 0, 1), (1, 4, 64, 1, 3, 2), (1, 40, 100, 2000, 9, 3),
    (3, 5, 300, 1, 5, 4), (8, 16, 900, 1, 4, 5), (64, 16, 960, 1, 20, 6), (64, 16, 960, 60, 3, 7),
    (257, 9, 500, 20, 50, 8), (1500, 6, 300, 12, 900, 9), (4096, 3, 180, 2, 0, 10),
    (5, 700, 40000, 4000, 30, 11),
])
def test_plan(dev, R, width, longest, n_new, spare, seed):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, longest + 1, R)
    new = rng.integers(0, n_new + 1, R)
    new[0] = n_new
    table, free, state = ref.tables(lens, width, int((-(-lens // 64)).sum()) + spare + 1, rng)
    check_plan(dev, table, lens, new, free, state, int(new.sum()))


@pytest.mark.parametrize("rows", [0, 1, 130, 400, 10000])
def test_plan_rows_fewer_and_more_than_asked(dev, rows):
    """Rows run out in the middle of a request; rows behind the last request
    have no slot."""
    rng = np.random.default_rng(3)
    lens, new = rng.integers(0, 200, 9), rng.integers(0, 90, 9)
    table, free, state = ref.tables(lens, 8, 80, rng)
    check_plan(dev, table, lens, new, free, state, rows, stride=11)


def test_plan_blocks_run_out(dev):
    """The free list ends inside a request; later ones still fill the blocks
    that they have."""
    lens, new = np.array([10, 64, 100, 130, 0]), np.array([200, 10, 70, 40, 3])
    for spare in range(8):
        table, free, state = ref.tables(lens, 6, 7 + spare, np.random.default_rng(spare))
        check_plan(dev, table, lens, new, free, state, 323)


def test_plan_tables_end_and_odd_lengths(dev):
    """Lengths up to and past what the table holds, negative ones, idle
    requests, a free count outside the list."""
    rng = np.random.default_rng(5)
    lens, new = np.array([128, 120, 127, 0, 5]), np.array([3, 20, 1, 0, -4])
    table, free, state = ref.tables(lens, 2, 12, rng)
    check_plan(dev, table, lens, new, free, state, 24)
    check_plan(dev, table, lens, new, free, np.array([-3, 0]), 24)
    t, p = run_plan(dev, table, np.array([900, -7, 64, 0, 5]), np.array([1, 2, 1, 0, 2 ** 31 - 1]),
                    free, state, 24)
    assert host(p.lens).tolist() == [128, 2, 65, 0, 25]
    # 1 + 2 + 1 + (2^31 - 1) asked, 2 + 1 + 20 stored
    assert host(p.slots)[0] == -1 and host(p.state)[1] == 2 ** 31 + 3 - 23


def test_plan_under_a_graph(dev):
    """One captured step, replayed for step after step on lengths in place."""
    rng = np.random.default_rng(1)
    R = 7
    lens = rng.integers(0, 100, R)
    table, free, state = ref.tables(lens, 4, 40, rng)
    t, l, f, s = (dev_i32(a, dev) for a in (table, lens, free, state))
    new = torch.ones(R, dtype=torch.int32, device=dev)
    plan = ops.kv_plan(t.clone(), l, new, f, s, R)
    plan = ops.KVPlan(*(torch.zeros_like(x) for x in plan))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv_plan(t, l, new, f, s, R, out=plan)
        l.copy_(plan.lens)
        s.copy_(plan.state)
    ones = np.ones(R, dtype=np.int64)
    for _ in range(70):
        g.replay()
        table, slots, positions, chunks, lens, state = ref.plan(table, lens, ones, free, state, R)
        for a, b in zip((t, *plan, l), (table, slots, positions, chunks, lens, state, lens)):
            assert np.array_equal(host(a), b)


def test_release(dev):
    rng = np.random.default_rng(2)
    for R, width, longest in ((1, 1, 0), (5, 4, 200), (300, 5, 300), (40, 150, 9000)):
        lens = rng.integers(0, longest + 1, R)
        used = int((-(-lens // 64)).sum())
        table, free, state = ref.tables(lens, width, used + 7, rng)
        t, l, f, s = (dev_i32(a, dev) for a in (table, lens, free, state))
        done = rng.integers(0, 2, R)
        ops.kv_release(t, l, dev_i32(done, dev), f, s)
        given = [b for r in range(R) if done[r] for b in table[r] if b >= 0]
        assert host(s)[0] == 7 + len(given)
        assert host(f)[7:7 + len(given)].tolist() == given
        assert np.array_equal(host(l), np.where(done, 0, lens))
        assert np.array_equal(host(t), np.where(done[:, None] > 0, -1, table))


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
def random_cache(n_blocks, Hk, D, rng):
    k = rng.integers(-127, 128, (n_blocks, Hk, 64, D)).astype(np.int8)
    v = rng.integers(-127, 128, (n_blocks, Hk, D, 64)).astype(np.int8)
    ks, vs = (rng.uniform(0.005, 0.03, (n_blocks, Hk)).astype(np.float32) for _ in range(2))
    return k, v, ks, vs


def step(dev, lens, new, width, spare, rng, rows=None):
    """A planned step: (plan on the GPU, table on the GPU, the reference's plan)."""
    lens, new = np.array(lens), np.array(new)
    n_blocks = int((-(-(lens + new) // 64)).sum()) + spare
    table, free, state = ref.tables(lens, width, n_blocks, rng)
    n = int(new.sum()) if rows is None else rows
    t, p = check_plan(dev, table, lens, new, free, state, n)
    return p, t, ref.plan(table, lens, new, free, state, n), n_blocks, n


def angles(n, D):
    a = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


APPENDS = [
    # lens, new, heads, kv heads, head dim
    ([0], [1], 1, 1, 16), ([5], [1], 2, 1, 64), ([63, 64, 0], [1, 1, 1], 4, 4, 128),
    ([0, 130, 7], [64, 0, 200], 4, 2, 80), ([1, 62], [63, 70], 6, 2, 96), ([30], [300], 3, 3, 256),
    ([10, 20, 90, 0], [3, 33, 1, 128], 8, 1, 48), ([17], [40], 20, 20, 128), ([3, 9], [31, 2], 2, 2, 112),
    ([10, 0], [150, 33], 8, 1, 256), ([61], [200], 32, 4, 64),
]


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(dev, case, dt):
    lens, new, H, Hk, D = APPENDS[case]
    rng = np.random.default_rng(case)
    p, t, want, n_blocks, n = step(dev, lens, new, 8, 2, rng, rows=sum(new) + 2)
    cache = random_cache(n_blocks, Hk, D, rng)
    # rows of very different size, so that some blocks' scales grow and some do
    # not; some rows zero
    size = 10.0 ** rng.uniform(-3, 1, (n, 1)) * (rng.random((n, 1)) > 0.1)
    x = torch.from_numpy((rng.standard_normal((n, (H + 2 * Hk) * D)) * size).astype(np.float32))
    x = x.to(DT[dt])
    cos, sin = angles(600, D)
    mine = [a.copy() for a in cache]
    q = ref.append(x.float().numpy(), want[1], want[2], want[3], cos, sin, *mine, H)
    gpu = [torch.from_numpy(a).to(dev) for a in cache]
    out = torch.full((n, H * D), 5.0, dtype=DT[dt], device=dev)
    ops.kv8_append(x.to(dev), p, torch.from_numpy(cos).to(dev), torch.from_numpy(sin).to(dev), *gpu,
                   H, q=out)
    for name, a, b in zip(("k", "v", "k_scale", "v_scale"), gpu, mine):
        assert np.array_equal(host(a), b), name
    got = host(out.float()).reshape(n, H, D)
    empty = want[1] < 0
    assert empty.sum() == 2 and (got[empty] == 5).all()
    # two products and a sum, then the factor and its rounding: 5 roundings of
    # at most |a| + |b| <= 2^0.5 of the pair's size; the output's own in bf16
    pair = np.abs(x.float().numpy()).reshape(n, -1)[:, :H * D].reshape(n, H, D // 2, 2).sum(-1)
    bound = 5 * 2.0 ** -24 * pair.repeat(2, -1).reshape(n, H, D) / math.sqrt(D)
    bound = bound + (2.0 ** -8 * np.abs(q) if dt == "bf16" else 0)
    assert (np.abs(got - q)[~empty] <= bound[~empty]).all()
    # the same through a strided, unaligned view
    again = [torch.from_numpy(a).to(dev) for a in cache]
    wide = torch.zeros(n, x.shape[1] + 5, dtype=DT[dt], device=dev)
    wide[:, 3:-2] = x.to(dev)
    out2 = torch.full((n, H * D + 7), 5.0, dtype=DT[dt], device=dev)
    ops.kv8_append(wide[:, 3:-2], p, torch.from_numpy(cos).to(dev), torch.from_numpy(sin).to(dev),
                   *again, H, q=out2[:, 1:-6])
    assert all(torch.equal(a, b) for a, b in zip(gpu, again))
    assert torch.equal(out2[:, 1:-6], out) and (out2[:, 0] == 5).all() and (out2[:, -6:] == 5).all()


def test_append_token_by_token_and_read(dev):
    """A request fed token by token: after each, every cached key and value is
    within half a step (its block's scale) for each time its block's scale grew,
    and once more for its own rounding."""
    rng = np.random.default_rng(4)
    H = Hk = 2
    D, n = 64, 150
    cos, sin = angles(n, D)
    x = rng.standard_normal((n, 3 * H * D)).astype(np.float32) * np.linspace(0.2, 3, n)[:, None].astype(np.float32)
    keys = ref.rope(x[:, H * D:2 * H * D].reshape(n, H, D), cos[:, None], sin[:, None])
    values = x[:, 2 * H * D:].reshape(n, H, D)
    gpu = [torch.from_numpy(a).to(dev) for a in random_cache(3, Hk, D, rng)]
    table = torch.full((1, 3), -1, dtype=torch.int32, device=dev)
    lens, state = (torch.tensor(a, dtype=torch.int32, device=dev) for a in ([0], [3, 0]))
    free, one = (torch.tensor(a, dtype=torch.int32, device=dev) for a in ([2, 0, 1], [1]))
    c, s = torch.from_numpy(cos).to(dev), torch.from_numpy(sin).to(dev)
    xd = torch.from_numpy(x).to(dev)
    for i in range(n):
        p = ops.kv_plan(table, lens, one, free, state, 1)
        ops.kv8_append(xd[i:i + 1], p, c, s, *gpu, H)
        lens, state = p.lens, p.state
    assert host(table).tolist() == [[1, 0, 2]]
    slots = torch.tensor([b * 64 + i for b in (1, 0, 2) for i in range(64)][:n], dtype=torch.int32,
                         device=dev)
    got_k, got_v = ops.kv8_read(slots, *gpu)
    for got, want in ((got_k, keys), (got_v, values)):
        for b in range(3):
            rows = slice(64 * b, min(64 * b + 64, n))
            peak = np.maximum.accumulate(np.abs(want[rows]).max(-1), 0)   # (token, head)
            grew = (np.diff(peak, axis=0) > 0).sum(0) + 1
            step = peak[-1] / 127
            err = np.abs(host(got)[rows] - want[rows]).max((0, 2))
            assert (err <= (0.5 * grew + 0.01) * step).all()


def test_append_infinite_and_position_past_tables(dev):
    """A NaN or infinity leaves its own block and head NaN and no other; so
    does a position without angles, its queries too."""
    rng = np.random.default_rng(6)
    p, t, want, n_blocks, n = step(dev, [10, 60], [4, 20], 2, 1, rng)
    H, Hk, D = 2, 2, 32
    for bad, column in ((math.inf, 2 * D + 5), (-math.inf, 3 * D + 1), (math.nan, 4 * D), (math.nan, 5 * D + 31)):
        cache = random_cache(n_blocks, Hk, D, rng)
        x = rng.standard_normal((n, 6 * D)).astype(np.float32)
        x[6, column] = bad          # request 1's third row: its first block
        cos, sin = angles(100, D)
        gpu = [torch.from_numpy(a).to(dev) for a in cache]
        mine = [a.copy() for a in cache]
        args = [torch.from_numpy(a).to(dev) for a in (cos, sin)]
        ops.kv8_append(torch.from_numpy(x).to(dev), p, *args, *gpu, H)
        with np.errstate(all="ignore"):
            ref.append(x, want[1], want[2], want[3], cos, sin, *mine, H)
        for a, b in zip(gpu, mine):
            assert np.array_equal(host(a), b)
        keys, values = (host(a) for a in ops.kv8_read(p.slots, *gpu))
        which = np.zeros((n, 2, 2), dtype=bool)      # row, k / v, head
        which[4:8, (column // D - 2) // 2, column // D % 2] = True
        assert np.array_equal(np.isnan(keys).all(-1), which[:, 0])
        assert np.array_equal(np.isnan(values).all(-1), which[:, 1])
        assert np.array_equal(np.isnan(keys).any(-1), which[:, 0])
    gpu = [torch.from_numpy(a).to(dev) for a in random_cache(n_blocks, Hk, D, rng)]
    x = torch.from_numpy(rng.standard_normal((n, 6 * D)).astype(np.float32)).to(dev)
    q = ops.kv8_append(x, p, args[0][:64], args[1][:64], *gpu, H)
    past = host(p.positions) >= 64
    assert past.sum() == 16 and np.array_equal(np.isnan(host(q)).any(1), past)
    keys, values = (host(a) for a in ops.kv8_read(p.slots, *gpu))
    assert np.array_equal(np.isnan(keys).any((1, 2)), past) and np.isfinite(values).all()


def test_append_slots_outside_the_cache(dev):
    """Slots past the cache and chunks past the rows touch nothing."""
    rng = np.random.default_rng(7)
    gpu = [torch.from_numpy(a).to(dev) for a in random_cache(2, 1, 16, rng)]
    keep = [a.clone() for a in gpu]
    cos, sin = (torch.from_numpy(a).to(dev) for a in angles(64, 16))
    x = torch.ones(4, 48, device=dev)

    def plan(slots, chunks):
        return ops.KVPlan(*(torch.tensor(a, dtype=torch.int32, device=dev)
                            for a in (slots, [0, 1, 2, 3], chunks, [4], [0, 0])))
    for slots, chunks in (([128] * 4, [[0, 4, 0, 0]]), ([0, 1, 2, 3], [[1, 4, 0, 0], [-1, 2, 0, 0]]),
                          ([62, 63, 64, 65], [[0, 4, 0, 0]]), ([-1] * 4, [[0, 4, 0, 0]]),
                          ([0, 1, 2, 3], [[0, 0, 0, 0], [0, -3, 0, 0], [0, 65, 0, 0], [4, 1, 0, 0]])):
        ops.kv8_append(x, plan(slots, chunks), cos, sin, *gpu, 1)
        assert all(torch.equal(a, b) for a, b in zip(gpu, keep))


@pytest.mark.parametrize("Hk,D,n", [(1, 16, 1), (3, 80, 64), (2, 256, 65), (20, 128, 200)])
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_read(dev, Hk, D, n, dt):
    rng = np.random.default_rng(n)
    cache = random_cache(5, Hk, D, rng)
    k, v, ks, vs = cache
    slots = rng.integers(-1, 5 * 64 + 3, n)
    slots[0] = 64
    keys, values = ops.kv8_read(dev_i32(slots, dev), *(torch.from_numpy(a).to(dev) for a in cache),
                                dtype=DT[dt])
    ok = (slots >= 0) & (slots < 320)
    b, i = np.where(ok, slots, 0) // 64, np.where(ok, slots, 0) % 64
    for got, want in ((keys, k[b, :, i] * ks[b][..., None]), (values, v[b, :, :, i] * vs[b][..., None])):
        want = torch.from_numpy(np.where(ok[:, None, None], want, 0).astype(np.float32)).to(DT[dt])
        assert torch.equal(got.cpu(), want)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
ATTENTION = [
    # lens, new, heads, kv heads, head dim
    ([0], [1], 1, 1, 16), ([0, 62, 63, 64, 300], [1] * 5, 4, 4, 128), ([200, 0], [1, 1], 20, 20, 128),
    ([0], [64], 2, 2, 64), ([0, 5], [130, 77], 3, 3, 128), ([100], [17], 8, 2, 96),
    ([70, 0, 1], [3, 9, 100], 16, 2, 80), ([500, 20], [1, 40], 10, 1, 256), ([33], [70], 5, 5, 32),
    ([1000, 7], [1, 1], 32, 2, 64), ([127], [65], 6, 3, 112), ([64] * 9, [1] * 9, 64, 1, 128),
]
RULES = {"plain": {}, "capped": {"softcap": 5.0}, "window": {"window": 50}, "one": {"window": 1},
         "slopes": {"slopes": True}, "prefix": {"prefix": True},
         "all": {"softcap": 20.0, "window": 70, "slopes": True, "prefix": True}}


def check_attention(dev, p, t, want, q, cache, H, out_dt, rules, rng, fill=5.0):
    table, slots, _, chunks, lens, _ = want
    R, n, D = len(lens), len(slots), cache[0].shape[3]
    kw, mine = dict(rules), dict(rules)
    if rules.get("slopes"):
        mine["slopes"] = (2.0 ** -rng.uniform(0.5, 8, H)).astype(np.float32)
        kw["slopes"] = torch.from_numpy(mine["slopes"]).to(dev)
    if rules.get("prefix"):
        mine["prefix"] = (rng.random(R) * (lens + 20)).astype(np.int64)
        kw["prefix"] = dev_i32(mine["prefix"], dev)
    out = torch.full((n, H * D), fill, dtype=DT[out_dt], device=dev)
    gpu = [torch.from_numpy(a).to(dev) for a in cache]
    ops.kv8_attention(q.to(dev), p, t, *gpu, out=out, **kw)
    exact, loss, top = ref.attention(q.float().numpy(), chunks, table, *cache, lens, **mine)
    got = host(out.float()).reshape(n, H, D)
    empty = slots < 0
    assert (got[empty] == fill).all()
    got, exact, loss, top = (a[~empty] for a in (got, exact, loss, top))
    # exponents: q's digits (u of its largest times the sum of |k|) and ten fp32
    # roundings of sums and factors, twice (numerator and denominator); weights:
    # u of their block's largest each, 64 a block; two of exp2, three a block of
    # the running sums, ten at the end
    u = 2.0 ** -24 if out_dt == "fp32" else 2.0 ** -16
    blocks = 1 + int(lens.max()) // 64
    rel = 2 * (u + 10 * 2.0 ** -24) * loss + 64 * u + (14 + 3 * blocks) * 2.0 ** -24
    bound = (rel * top)[..., None] + (2.0 ** -8 * np.abs(exact) if out_dt == "bf16" else 0)
    assert np.isfinite(got).all()
    worst = (np.abs(got - exact) / (bound + 1e-30)).max()
    assert worst <= 1, worst
    return kw, gpu, out


@pytest.mark.parametrize("rules", sorted(RULES))
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(dev, case, dt, rules):
    lens, new, H, Hk, D = ATTENTION[case]
    rng = np.random.default_rng(case)
    p, t, want, n_blocks, n = step(dev, lens, new, 18, 2, rng, rows=sum(new) + 1)
    cache = random_cache(n_blocks, Hk, D, rng)
    q = rng.standard_normal((n, H * D)) * D ** -0.5 * rng.uniform(0.2, 4, (n, 1))
    q = torch.from_numpy(q.astype(np.float32)).to(DT[dt])
    kw, gpu, out = check_attention(dev, p, t, want, q, cache, H, dt, RULES[rules], rng)
    # strided, unaligned queries and outputs: the same bits
    wide = torch.zeros(n, H * D + 3, dtype=DT[dt], device=dev)
    wide[:, 1:-2] = q.to(dev)
    out2 = torch.full((n, H * D + 3), 5.0, dtype=DT[dt], device=dev)
    ops.kv8_attention(wide[:, 1:-2], p, t, *gpu, out=out2[:, 2:-1], **kw)
    assert torch.equal(out2[:, 2:-1], out) and (out2[:, :2] == 5).all() and (out2[:, -1] == 5).all()


@pytest.mark.parametrize("dt,out_dt", [("fp32", "bf16"), ("bf16", "fp32")])
def test_attention_mixed_types(dev, dt, out_dt):
    rng = np.random.default_rng(1)
    p, t, want, n_blocks, n = step(dev, [90, 0], [1, 20], 4, 2, rng)
    cache = random_cache(n_blocks, 2, 64, rng)
    q = torch.from_numpy(rng.standard_normal((n, 256)).astype(np.float32) * 0.2).to(DT[dt])
    check_attention(dev, p, t, want, q, cache, 4, out_dt, {}, rng)


@pytest.mark.parametrize("rules", ["plain", "window", "prefix", "all"])
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("lens,new,H,Hk,D", [([5000, 40, 0], [1, 1, 1], 4, 2, 128), ([9000], [2], 6, 1, 64),
                                             ([4100, 3000], [1, 3], 2, 2, 256)])
def test_attention_split_over_long_caches(dev, lens, new, H, Hk, D, dt, rules):
    """Few rows over wide tables: several workgroups to a row, joined."""
    rng = np.random.default_rng(7)
    p, t, want, n_blocks, n = step(dev, lens, new, 160, 2, rng, rows=sum(new) + 1)
    cache = random_cache(n_blocks, Hk, D, rng)
    q = torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32) * 2 * D ** -0.5).to(DT[dt])
    kw = {k: (v if k != "window" else 700) for k, v in RULES[rules].items()}
    from nativebit_amd import _lib
    assert _lib.load().nb_kv8_attention_ws_bytes(n, p.chunks.shape[0], 160, H, Hk, D) > 0
    check_attention(dev, p, t, want, q, cache, H, dt, kw, rng)


def test_attention_sharp_and_flat_rows(dev):
    """Rows whose largest score is far ahead, rows of zeros, rows of values
    below 2^-100, blocks of scale 0 and scales far apart."""
    rng = np.random.default_rng(3)
    H = Hk = 3
    D = 64
    p, t, want, n_blocks, n = step(dev, [400, 100], [40, 1], 8, 2, rng)
    cache = list(random_cache(n_blocks, Hk, D, rng))
    cache[2][::2] *= 1e-3
    cache[3] = (cache[3] * 10.0 ** rng.integers(-6, 3, cache[3].shape)).astype(np.float32)
    cache[2][1] = cache[3][2] = 0
    q = rng.standard_normal((n, H * D)).astype(np.float32)
    q[:10] *= 30
    q[10:20] = 0
    q[20:25] *= np.float32(1e-36)
    q[25:30, ::3] *= np.float32(1e-4)
    check_attention(dev, p, t, want, torch.from_numpy(q), cache, H, "fp32", {}, rng)


def test_attention_tables_with_holes(dev):
    """Blocks outside the cache are not seen; a row that sees nothing is 0."""
    rng = np.random.default_rng(5)
    p, t, want, n_blocks, n = step(dev, [300, 20, 700], [1, 2, 70], 13, 2, rng)
    table = want[0]
    table[0, 1], table[0, 3], table[1, 0], table[2, 4:9] = -1, n_blocks, -5, 2 ** 30
    t.copy_(dev_i32(table, dev))
    cache = random_cache(n_blocks, 2, 64, rng)
    q = torch.from_numpy(rng.standard_normal((n, 256)).astype(np.float32) * 0.3)
    for rules in ({}, {"window": 90}, {"prefix": True}):
        _, _, out = check_attention(dev, p, t, want, q, cache, 4, "fp32", rules, rng)
        assert (out[1:3] == 0).all()


def test_attention_poisoned_blocks_and_queries(dev):
    """NaN stays with the rows that see it: a block of scale inf (codes 0, as
    an append leaves it), a NaN or infinite query row."""
    rng = np.random.default_rng(6)
    lens, new, H, D = [130, 64], [70, 3], 2, 64
    p, t, want, n_blocks, n = step(dev, lens, new, 6, 2, rng)
    cache = [torch.from_numpy(a).to(dev) for a in random_cache(n_blocks, H, D, rng)]
    q = torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32) * 0.2).to(dev)
    clean = ops.kv8_attention(q, p, t, *cache)
    last = int(want[0][0, 3])     # request 0: positions 192 .. 199, rows 62 .. 69
    for code, scale in ((0, 2), (1, 3)):
        bad = [a.clone() for a in cache]
        bad[code][last, 1] = 0
        bad[scale][last, 1] = math.inf
        out = ops.kv8_attention(q, p, t, *bad)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[62:70, D:] = True
        assert torch.equal(torch.isnan(out), hit)
        assert torch.equal(out[~hit], clean[~hit])
        # out of the window of later rows, it is not seen
        for w in (1, 5):
            near = ops.kv8_attention(q, p, t, *bad, window=w)
            assert torch.equal(torch.isnan(near), hit)
    for value in (math.nan, math.inf, -math.inf):
        q2 = q.clone()
        q2[5, 3] = value
        out = ops.kv8_attention(q2, p, t, *cache)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[5, :D] = True
        assert torch.equal(torch.isnan(out), hit) and torch.equal(out[~hit], clean[~hit])


def test_attention_stale_slots_are_not_read(dev):
    """What the unused slots of a block hold changes nothing."""
    rng = np.random.default_rng(8)
    p, t, want, n_blocks, n = step(dev, [70, 3], [2, 30], 6, 2, rng)
    cache = [torch.from_numpy(a).to(dev) for a in random_cache(n_blocks, 2, 128, rng)]
    q = torch.from_numpy(rng.standard_normal((n, 512)).astype(np.float32) * 0.2).to(dev)
    out = ops.kv8_attention(q, p, t, *cache)
    for r, end in enumerate((72, 33)):
        b = int(want[0][r, end // 64])
        cache[0][b, :, end % 64:] = 127
        cache[1][b, :, :, end % 64:] = -127
    unused = [b for b in range(n_blocks) if b not in want[0]]
    for a in cache[2:]:
        a[unused] = math.nan
    assert torch.equal(ops.kv8_attention(q, p, t, *cache), out)


def test_attention_far_blocks(dev):
    """Blocks beyond 2^31 bytes of codes."""
    Hk, D = 8, 128
    n_blocks = 2 ** 31 // (Hk * 64 * D) + 40
    rng = np.random.default_rng(9)
    k = torch.zeros(n_blocks, Hk, 64, D, dtype=torch.int8, device=dev)
    v = torch.zeros(n_blocks, Hk, D, 64, dtype=torch.int8, device=dev)
    ks, vs = torch.zeros(n_blocks, Hk, device=dev), torch.zeros(n_blocks, Hk, device=dev)
    lens, new = np.array([100]), np.array([30])
    far = [n_blocks - 1, n_blocks - 30, n_blocks - 2]
    state = np.array([3, 0])
    free = np.zeros(n_blocks, dtype=np.int32)
    free[:3] = far[::-1]
    table = torch.full((1, 4), -1, dtype=torch.int32, device=dev)
    f, s = dev_i32(free, dev), dev_i32(state, dev)
    cos, sin = (torch.from_numpy(a).to(dev) for a in angles(200, D))
    x = torch.randn(130, 3 * Hk * D, device=dev, generator=torch.Generator(dev).manual_seed(1))
    p1 = ops.kv_plan(table, dev_i32([0], dev), dev_i32(lens, dev), f, s, 100)
    ops.kv8_append(x[:100], p1, cos, sin, k, v, ks, vs, Hk)
    p2 = ops.kv_plan(table, p1.lens, dev_i32(new, dev), f, p1.state, 30)
    q = ops.kv8_append(x[100:], p2, cos, sin, k, v, ks, vs, Hk)
    assert host(table)[0, :3].tolist() == far
    out = ops.kv8_attention(q, p2, table, k, v, ks, vs)
    small = torch.tensor([[0, 1, 2, -1]], dtype=torch.int32, device=dev)
    near = [a[far].contiguous() for a in (k, v, ks, vs)]
    assert torch.equal(out, ops.kv8_attention(q, p2, small, *near))
    keys, values = ops.kv8_read(p2.slots, k, v, ks, vs)
    slots = (p2.positions % 64 + 64 * (p2.positions // 64)).int()
    for a, b in zip((keys, values), ops.kv8_read(slots, *near)):
        assert torch.equal(a, b) and a.abs().sum() > 0


# ---------------------------------------------------------------------------
# rules on logits
# ---------------------------------------------------------------------------
def logits_inputs(B, V, n, dt, rng):
    x = torch.from_numpy((rng.standard_normal((B, V)) * 4).astype(np.float32)).to(DT[dt])
    history = rng.integers(-2, V + 3, (B, n))
    history[:, ::2] = rng.integers(0, min(V, 7), history[:, ::2].shape)    # repeated tokens
    lens = rng.integers(-1, n + 2, B)
    ids = rng.integers(-1, V + 1, (B, 9))
    ids[:, 5] = ids[:, 2]                                              # listed twice
    return {"x": x, "history": history, "lens": lens, "prompt": (lens * rng.random(B)).astype(np.int64),
            "repetition": rng.uniform(0.7, 1.5, B).astype(np.float32),
            "frequency": rng.uniform(-0.3, 0.6, B).astype(np.float32),
            "presence": rng.uniform(-0.3, 0.6, B).astype(np.float32), "ids": ids,
            "bias": (rng.standard_normal((B, 9)) * 3).astype(np.float32),
            "mask": rng.integers(-2 ** 31, 2 ** 31, (B, (V + 31) // 32))}


NAMES = {"prompt": "prompt_lens", "ids": "bias_ids"}


def run_logits(dev, d, use, **kw):
    a = {}
    for name in use:
        t = d[name]
        a[NAMES.get(name, name)] = dev_i32(t, dev) if t.dtype.kind == "i" else torch.from_numpy(t).to(dev)
    return ops.logits_rules(d["x"].to(dev), choose=True, **a, **kw)


@pytest.mark.parametrize("use", [
    (), ("history", "lens", "repetition"), ("history", "lens", "frequency", "presence"),
    ("ids", "bias"), ("mask",),
    ("history", "lens", "prompt", "repetition", "frequency", "presence", "ids", "bias", "mask")])
@pytest.mark.parametrize("B,V,n,dt", [(1, 1, 1, "fp32"), (3, 37, 20, "bf16"), (2, 4096, 300, "fp32"),
                                      (5, 4097, 65, "bf16"), (3, 9001, 0, "fp32"), (2, 12290, 700, "fp32")])
def test_logits(dev, B, V, n, dt, use):
    d = logits_inputs(B, V, n, dt, np.random.default_rng(V))
    want, chosen = ref.rules(d["x"].float().numpy(), **{k: d[k] for k in use})
    out, tokens = run_logits(dev, d, use)
    assert np.array_equal(host(out), want) and np.array_equal(host(tokens), chosen)
    # one row at a time through views at odd places, and in place
    for b in range(B):
        wide = torch.zeros(B, V + 5, dtype=DT[dt], device=dev)
        wide[:, 2:V + 2] = d["x"].to(dev)
        one = {k: (v[b:b + 1] if k != "x" else wide[b:b + 1, 2:V + 2]) for k, v in d.items()}
        o = torch.empty(1, V + 3, device=dev)
        got, token = run_logits(dev, one, use, out=o[:, 1:V + 1])
        assert np.array_equal(host(got)[0], want[b]) and host(token)[0] == chosen[b]
        if dt == "fp32":
            got, _ = run_logits(dev, one, use, out=one["x"])
            assert got.data_ptr() == one["x"].data_ptr() and np.array_equal(host(got)[0], want[b])
            assert (wide[:, :2] == 0).all() and (wide[:, V + 2:] == 0).all()


def test_logits_ties_and_nothing_left(dev):
    V = 9000
    x = torch.zeros(8, V, device=dev)
    x[0, [700, 8000]] = 3.0                     # a tie across workgroups
    x[1, :] = -math.inf
    x[2, :] = math.nan
    x[3, 5] = math.nan                          # passed over
    x[4, :] = -math.inf
    x[4, 8999] = -3.4e38
    x[5, 100], x[5, 4000] = math.inf, math.inf
    x[6, :] = -1.0
    x[6, 17], x[6, 3], x[6, 4] = -0.0, 0.0, -2.0   # zeros are equal
    mask = torch.full((8, (V + 31) // 32), -1, dtype=torch.int32, device=dev)
    mask[7] = 0
    out, tokens = ops.logits_rules(x, mask=mask, choose=True)
    assert host(tokens).tolist() == [700, -1, -1, 0, 8999, 100, 3, -1]
    assert torch.equal(out[:7].nan_to_num(7), x[:7].nan_to_num(7)) and (out[7] == -math.inf).all()


def test_logits_shared_rules(dev):
    """One history, bias list and mask for all rows (row stride 0)."""
    rng = np.random.default_rng(2)
    d = logits_inputs(4, 5000, 50, "fp32", rng)
    for name in ("history", "ids", "bias", "mask"):
        d[name] = np.repeat(d[name][:1], 4, 0)
    use = [k for k in d if k != "x"]
    want, chosen = ref.rules(d["x"].numpy(), **{k: d[k] for k in use})
    a = {NAMES.get(k, k): (dev_i32(d[k], dev) if d[k].dtype.kind == "i" else
                           torch.from_numpy(d[k]).to(dev)) for k in use}
    for name in ("history", "bias_ids", "bias", "mask"):
        a[name] = a[name][:1].expand(4, -1)
    out, tokens = ops.logits_rules(d["x"].to(dev), choose=True, **a)
    assert np.array_equal(host(out), want) and np.array_equal(host(tokens), chosen)


# ---------------------------------------------------------------------------
# streams and graphs
# ---------------------------------------------------------------------------
def test_step_under_graphs_and_streams(dev):
    """A step's operators captured twice and replayed in turn and on another
    stream, against the eager results each time."""
    rng = np.random.default_rng(11)
    H, Hk, D, V = 8, 2, 128, 6000
    p, t, want, n_blocks, n = step(dev, [4200, 10, 500], [1, 1, 1], 70, 2, rng)
    cache = random_cache(n_blocks, Hk, D, rng)
    cos, sin = (torch.from_numpy(a).to(dev) for a in angles(5000, D))
    w = torch.randn(H * D, V, device=dev, generator=torch.Generator(dev).manual_seed(2)) * 0.1
    hist = dev_i32(rng.integers(0, V, (3, 40)), dev)
    lens = dev_i32([40, 3, 0], dev)
    rep = torch.full((3,), 1.3, device=dev)
    caches = [[torch.from_numpy(a).to(dev) for a in cache] for _ in range(3)]
    xs = [torch.zeros(n, (H + 2 * Hk) * D, device=dev) for _ in range(2)]

    def work(x, c):
        q = ops.kv8_append(x, p, cos, sin, *c, H)
        att = ops.kv8_attention(q, p, t, *c)
        out, tokens = ops.logits_rules(att @ w, history=hist, lens=lens, repetition=rep, choose=True)
        return att, out, tokens
    graphs, results = [], []
    for x, c in zip(xs, caches):
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            work(x, c)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(work(x, c))
        graphs.append(g)
    side = torch.cuda.Stream(dev)
    for i in range(6):
        for j, (g, x) in enumerate(zip(graphs, xs)):
            x.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)))
            for a, b in zip(caches[j], cache):
                a.copy_(torch.from_numpy(b))
            for a, b in zip(caches[2], cache):
                a.copy_(torch.from_numpy(b))
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
                g.replay()
            torch.cuda.current_stream().wait_stream(side)
            eager = work(x, caches[2])
            for a, b in zip(results[j], eager):
                assert torch.equal(a, b)
            for a, b in zip(caches[j], caches[2]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("rules", ["plain", "all"])
def test_attention_split_prompts(dev, dt, rules):
    """Few chunks of many rows, some of few, over wide tables: split and
    joined row by row."""
    rng = np.random.default_rng(12)
    p, t, want, n_blocks, n = step(dev, [2100, 0, 700], [70, 1, 30], 40, 2, rng, rows=103)
    cache = random_cache(n_blocks, 2, 64, rng)
    q = torch.from_numpy(rng.standard_normal((n, 4 * 64)).astype(np.float32) * 0.3).to(DT[dt])
    from nativebit_amd import _lib
    assert _lib.load().nb_kv8_attention_ws_bytes(n, p.chunks.shape[0], 40, 4, 2, 64) > 0
    check_attention(dev, p, t, want, q, cache, 4, dt, RULES[rules], rng)


@pytest.mark.parametrize("lens,new,width,H,Hk,D", [
    ([130, 0, 700], [1, 1, 1], 18, 64, 1, 64),              # four tiles of rows a token
    ([130, 0, 700], [1, 0, 1], 18, 40, 1, 256),             # two and a half
    ([2100, 900], [1, 1], 40, 64, 1, 80),                   # split as well
    ([3] * 40 + [100] + [0] * 59, [0] * 40 + [90] + [0] * 59, 18, 4, 2, 128),
    ([3] * 40 + [2000] + [0] * 59, [1] * 40 + [47] + [0] * 59, 40, 8, 2, 64),
])
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("rules", ["plain", "all"])
def test_attention_many_rows_of_few_tokens(dev, lens, new, width, H, Hk, D, dt, rules):
    """No more tokens than requests, but chunks of many rows: many heads that
    share keys, one request that brings all tokens."""
    rng = np.random.default_rng(15)
    p, t, want, n_blocks, n = step(dev, lens, new, width, 2, rng)
    assert n <= len(lens)
    q = torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32) * 0.3).to(DT[dt])
    check_attention(dev, p, t, want, q, random_cache(n_blocks, Hk, D, rng), H, dt, RULES[rules], rng)


@pytest.mark.parametrize("lens,new,width,H,Hk,D", [
    ([30, 0, 700], [1, 1, 1], 18, 6, 2, 64),            # single tokens
    ([30, 5, 700], [200, 1, 70], 18, 6, 2, 64),         # prompts, codes shared
    ([2100, 0, 700], [1, 3, 1], 40, 4, 2, 128),         # split
    ([2100, 0, 700], [70, 1, 30], 40, 4, 2, 256),       # split prompts
])
@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_attention_in_place(dev, lens, new, width, H, Hk, D, dt):
    """out may be q, whole or columns of an array, and beside it in its rows."""
    rng = np.random.default_rng(13)
    p, t, want, n_blocks, n = step(dev, lens, new, width, 2, rng, rows=sum(new))
    cache = [torch.from_numpy(a).to(dev) for a in random_cache(n_blocks, Hk, D, rng)]
    q = torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32) * 0.3).to(DT[dt]).to(dev)
    out = ops.kv8_attention(q, p, t, *cache)
    both = torch.full((n, 2 * H * D + 8), 3.0, dtype=DT[dt], device=dev)
    both[:, :H * D] = q
    ops.kv8_attention(both[:, :H * D], p, t, *cache, out=both[:, H * D + 8:])
    assert torch.equal(both[:, :H * D], q) and torch.equal(both[:, H * D + 8:], out)
    ops.kv8_attention(both[:, :H * D], p, t, *cache, out=both[:, :H * D])
    assert torch.equal(both[:, :H * D], out) and bool((both[:, H * D:H * D + 8] == 3.0).all())
    assert ops.kv8_attention(q, p, t, *cache, out=q) is q and torch.equal(q, out)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_append_in_place(dev, dt):
    """q may be the query columns of qkv; the keys and values stay."""
    rng = np.random.default_rng(14)
    p, t, want, n_blocks, n = step(dev, [30, 0, 100], [70, 1, 3], 4, 2, rng, rows=74)
    H, Hk, D = 4, 2, 64
    qkv = torch.from_numpy(rng.standard_normal((n, (H + 2 * Hk) * D)).astype(np.float32)).to(DT[dt]).to(dev)
    a = torch.from_numpy(rng.uniform(0, 6, (256, D // 2)).astype(np.float32)).to(dev)
    first = [torch.from_numpy(x).to(dev) for x in random_cache(n_blocks, Hk, D, rng)]
    again, mine = [x.clone() for x in first], qkv.clone()
    q = ops.kv8_append(qkv, p, a.cos(), a.sin(), *first, H)
    ops.kv8_append(mine, p, a.cos(), a.sin(), *again, H, q=mine[:, :H * D])
    assert torch.equal(mine[:, :H * D], q) and torch.equal(mine[:, H * D:], qkv[:, H * D:])
    for x, y in zip(first, again):
        assert torch.equal(x, y)
