"""What nb_kv8_attention's fixed-point factors may lose, where the inputs spread
far: against 64 bits, with bounds in what a row really weighs (not in the
largest value that it sees)."""
import numpy as np
import pytest
import torch

from nativebit_amd import ops
from tests import serving_ref as ref
from tests.test_gpu_serving import DT, host, random_cache, step

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def weighed(q, want, cache, H, out_dt, scores=None):
    """(out, bound) in 64 bits of a step's rows over blocks that are taken two at
    a time from a request's first on.  With w the weights relative to the row's
    largest and W their sum, a pair of blocks whose largest w * v_scale is C
    loses of each weight half a step of C / (127 * 2^16) (bf16 outputs 127 * 2^8)
    and two roundings of the factor, and fp32 outputs half a unit of 2^-15 C of
    the sum; then come the scores' roundings, in the weights, and those of the
    running sums, both of sum w |v| / W."""
    table, slots, _, chunks, lens, _ = want
    k, v, ks, vs = cache
    Hk, D = k.shape[1], k.shape[3]
    n, G = q.shape[0], H // Hk
    out, bound = np.full((n, H, D), np.nan), np.full((n, H, D), np.nan)
    u = 2.0 ** -23 if out_dt == "fp32" else 2.0 ** -16
    for row0, count, r, pos0 in chunks:
        for t in range(row0, row0 + count):
            i = pos0 + t - row0
            ids = table[r, :i // 64 + 1]
            for h in range(H):
                g = h // G
                keys = (k[ids, g] * ks[ids, g].astype(np.float64)[:, None, None]).reshape(-1, D)[:i + 1]
                codes = v[ids, g].astype(np.float64).transpose(0, 2, 1).reshape(-1, D)[:i + 1]
                scale = np.repeat(vs[ids, g].astype(np.float64), 64)[:i + 1]
                x = q[t, h * D:(h + 1) * D].astype(np.float64)
                s = keys @ x
                size = np.abs(keys) @ np.abs(x) + np.abs(s)
                if scores is not None:
                    s = scores(s)
                w = np.exp(s - s.max())
                W = w.sum()
                out[t, h] = (w * scale) @ codes / W
                lost = np.zeros(D)
                for a in range(0, i + 1, 128):
                    part = slice(a, min(a + 128, i + 1))
                    C = (w[part] * scale[part]).max()
                    lost += C * (u * np.abs(codes[part]).sum(0) + (2.0 ** -16 if out_dt == "fp32" else 0))
                # (the scores' errors: 2 U a rounding of their terms, ten of them)
                rel = 2 * 10 * U * size.max() + (14 + 3 * len(ids)) * U + (0 if out_dt == "fp32" else 2.0 ** -16)
                bound[t, h] = lost / W + rel * (w * scale) @ np.abs(codes) / W
    return out, bound + (2.0 ** -8 * np.abs(out) if out_dt == "bf16" else 0)


def check(dev, p, t, want, q, cache, H, out_dt, **kw):
    exact, bound = weighed(q.float().numpy(), want, cache, H, out_dt, **kw)
    gpu = [torch.from_numpy(a).to(dev) for a in cache]
    out = ops.kv8_attention(q.to(dev), p, t, *gpu, out_dtype=DT[out_dt])
    ok = want[1] >= 0
    got = host(out.float()).reshape(exact.shape)
    assert np.isfinite(got[ok]).all()
    worst = (np.abs(got - exact) / (bound + 1e-30))[ok].max()
    assert worst <= 1, worst


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("large", [0, 1, 2])
@pytest.mark.parametrize("ratio", [16.0, 256.0, 4096.0, 1e5, 1e12, 1e30])
@pytest.mark.parametrize("D", [64, 256])
def test_scales_of_blocks_with_little_weight(dev, dt, large, ratio, D):
    """A prompt's rows weigh a block of far larger values with e^-30 (and less):
    its neighbour's weights keep their bits."""
    rng = np.random.default_rng(1)
    H = 2
    p, t, want, n_blocks, n = step(dev, [192], [60], 4, 1, rng)
    cache = random_cache(n_blocks, H, D, rng)
    k, v, ks, vs = cache
    ks[:], vs[:] = 0.01, 0.01
    block = want[0][0, large]
    vs[block] = 0.01 * ratio
    # one dim of q: scores of 0.5 a key code, 32 in the others' favour (their
    # codes exact in q's digits)
    k[:, :, :, 0] = rng.integers(50, 64, k.shape[:3])
    k[block, :, :, 0] -= 64 if ratio < 1e6 else 120
    q = np.zeros((n, H, D), dtype=np.float32)
    q[:, :, 0] = 50.0
    check(dev, p, t, want, torch.from_numpy(q.reshape(n, H * D)).to(DT[dt]), cache, H, dt)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_scales_of_blocks_at_random(dev, dt):
    """Value scales over twelve orders, weights over as many."""
    rng = np.random.default_rng(2)
    H, D = 3, 128
    p, t, want, n_blocks, n = step(dev, [500, 70], [70, 64], 12, 2, rng)
    k, v, ks, vs = random_cache(n_blocks, H, D, rng)
    vs = (vs * 10.0 ** rng.uniform(-6, 6, vs.shape)).astype(np.float32)
    q = rng.standard_normal((n, H * D)).astype(np.float32) * rng.uniform(0.05, 2, (n, 1)).astype(np.float32)
    q[:, D // 8:] = 0
    q[:, 2 * D:2 * D + 8] = 1
    check(dev, p, t, want, torch.from_numpy(q).to(torch.bfloat16).to(DT[dt]), (k, v, ks, vs), H, dt)


def test_blocks_of_infinite_scale_are_nan_in_pairs(dev):
    """Rows that see a poisoned block are NaN whatever its neighbour weighs."""
    rng = np.random.default_rng(3)
    H, D = 2, 64
    p, t, want, n_blocks, n = step(dev, [192], [60], 4, 1, rng)
    cache = [torch.from_numpy(a).to(dev) for a in random_cache(n_blocks, H, D, rng)]
    q = torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32)).to(dev)
    clean = ops.kv8_attention(q, p, t, *cache)
    for j in range(3):
        for scale in (torch.inf, torch.nan):
            bad = [a.clone() for a in cache]
            b = int(want[0][0, j])
            bad[1][b, 1], bad[3][b, 1] = 0, scale
            for weigh in (0, 100):     # its weights 1 or e^-large and below 2^-126
                bad[0][b, :] = cache[0][b, :] if not weigh else 0
                out = ops.kv8_attention(q, p, t, *bad)
                assert torch.isnan(out[:, D:]).all()
                if not weigh:
                    assert torch.equal(out[:, :D], clean[:, :D])


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("cap", [3.0, 255.0, 257.0, 1e4, 1e6, 1e8, 1e20])
@pytest.mark.parametrize("lens,new", [([70, 200], [60, 1]), ([70, 200, 3], [1, 1, 1])])
def test_caps_far_above_the_scores(dev, dt, cap, lens, new):
    """A cap's error goes by the score, not by the cap: 4e-7 of it (the tanh), for
    bf16 outputs and caps up to 256 2^-14 in the exponent besides."""
    rng = np.random.default_rng(4)
    H, Hk, D = 4, 2, 64
    p, t, want, n_blocks, n = step(dev, lens, new, 5, 1, rng)
    cache = random_cache(n_blocks, Hk, D, rng)
    q = torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32) * 0.4).to(DT[dt])
    gpu = [torch.from_numpy(a).to(dev) for a in cache]
    out = host(ops.kv8_attention(q.to(dev), p, t, *gpu, softcap=cap).float()).reshape(n, H, D)
    args = (q.float().numpy(), want[3], want[0], *cache, want[4])
    exact, _, top = ref.attention(*args, softcap=cap)
    _, loss, _ = ref.attention(*args)       # (the scores' sizes, without the cap's own term)
    u = U if dt == "fp32" else 2.0 ** -16
    blocks = 1 + int(want[4].max()) // 64
    rel = 2 * ((u + 17 * U) * loss + (2.0 ** -14 if dt == "bf16" and cap <= 256 else 0))
    rel = rel + 64 * u + (14 + 3 * blocks) * U
    bound = (rel * top)[..., None] + (2.0 ** -8 * np.abs(exact) if dt == "bf16" else 0)
    worst = (np.abs(out - exact) / bound).max()
    assert worst <= 1, worst


@pytest.mark.parametrize("dt,out_dt", [("fp32", "fp32"), ("bf16", "bf16"), ("fp32", "bf16"), ("bf16", "fp32")])
@pytest.mark.parametrize("large", [1.0, 30.0, 300.0, 3000.0, 1e5])
@pytest.mark.parametrize("lens,new,H,Hk,D", [([300], [70], 2, 2, 128), ([300, 40], [1, 1], 8, 2, 64),
                                             ([130], [40], 2, 1, 256), ([70], [1], 3, 3, 80)])
def test_rows_with_a_large_dim(dev, dt, out_dt, large, lens, new, H, Hk, D):
    """One dim of q far above the others, whose keys are small there: the others
    keep the bits that their scores need.  In rows whose largest value is over 8
    times their mean one an element loses 2^-32 of it (bf16 outputs 2^-24) beside
    its own rounding, in the others 2^-24 (2^-16); sums half a unit of 2^-15 of it
    but with 32 bits."""
    rng = np.random.default_rng(5)
    p, t, want, n_blocks, n = step(dev, lens, new, 7, 1, rng)
    cache = random_cache(n_blocks, Hk, D, rng)
    cache[0][:, :, :, 7] = rng.integers(-1, 2, cache[0].shape[:3])
    cache[2][:] = 0.02
    q = rng.standard_normal((n, H, D)).astype(np.float32) * np.float32(D ** -0.5)
    q[:, :, 7] *= np.float32(large)
    q = torch.from_numpy(q.reshape(n, H * D)).to(DT[dt])
    x = q.float().numpy().reshape(n, H, D).astype(np.float64)
    gpu = [torch.from_numpy(a).to(dev) for a in cache]
    out = host(ops.kv8_attention(q.to(dev), p, t, *gpu, out_dtype=DT[out_dt]).float()).reshape(n, H, D)
    exact, _, top = ref.attention(q.float().numpy(), want[3], want[0], *cache, want[4])
    table, blocks = want[0], 1 + int(want[4].max()) // 64
    fine = out_dt == "fp32"
    loss = np.zeros((n, H))
    for row0, count, r, pos0 in want[3]:
        for tok in range(row0, row0 + count):
            end = pos0 + tok - row0 + 1
            for h in range(H):
                g = h // (H // Hk)
                ids = table[r, :-(-end // 64)]
                k = np.abs(cache[0][ids, g].astype(np.float64) * 0.02).reshape(-1, D)[:end]
                peak = np.abs(x[tok, h]).max()
                spread = peak * D > 8.01 * np.abs(x[tok, h]).sum()
                # (a unit of the product's lower half, rounded to fp32: 2^-25)
                unit = peak * 0.02 * (2.0 ** -25 if fine and spread else 2.0 ** -16)
                digit = (2.0 ** -24 if fine else 2.0 ** -16) * (2.0 ** -8 if spread else 1)
                loss[tok, h] = (11 * U * k @ np.abs(x[tok, h]) + digit * peak * k.sum(1) + unit).max()
    u = U if fine else 2.0 ** -16
    rel = 2 * loss + 64 * u + (14 + 3 * blocks) * U
    bound = (rel * top)[..., None] + (0 if fine else 2.0 ** -8 * np.abs(exact))
    worst = (np.abs(out - exact) / bound).max()
    assert worst <= 1, worst


def test_rows_keep_their_result_beside_others(dev):
    """A row's result does not depend on what the rows of its tile need."""
    rng = np.random.default_rng(6)
    for lens, new, H, D in (([200], [70], 2, 128), ([200, 9], [1, 1], 16, 64)):
        p, t, want, n_blocks, n = step(dev, lens, new, 5, 1, rng)
        cache = [torch.from_numpy(a).to(dev) for a in random_cache(n_blocks, 1, D, rng)]
        q = torch.from_numpy(rng.standard_normal((n, H, D)).astype(np.float32)).to(dev)
        for out_dt in (torch.float32, torch.bfloat16):
            even = ops.kv8_attention(q.view(n, -1), p, t, *cache, out_dtype=out_dt).view(n, H, D)
            other = q.clone()
            other[0, 0, 3] = other[-1, 1, 5] = 1e4
            out = ops.kv8_attention(other.view(n, -1), p, t, *cache, out_dtype=out_dt).view(n, H, D)
            same = torch.ones(n, H, dtype=torch.bool, device=dev)
            same[0, 0] = same[-1, 1] = False
            assert torch.equal(out[same], even[same])
            assert not torch.equal(out, even)
