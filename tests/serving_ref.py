"""Plain restatements, in 64 bits or exact fp32 steps on the host, of the
serving operators (block tables, 8-bit cache, attention over it, rules on
logits)."""
import math

import numpy as np

BLOCK = 64


def plan(table, lens, new, free, state, n_tokens):
    """The allocator token by token: every token of every request in order
    asks for its slot.  Returns (table, slots, positions, chunks, lens, state)."""
    table, free = table.copy(), list(free[:max(0, min(int(state[0]), len(free)))])
    n_blocks = None
    R, width = table.shape
    slots, positions = np.full(n_tokens, -1), np.zeros(n_tokens, dtype=np.int64)
    ends, dropped, row = np.zeros(R, dtype=np.int64), 0, 0
    runs = []
    for r in range(R):
        n = end = max(0, min(int(lens[r]), width * BLOCK))
        full = False
        for i in range(max(0, int(new[r]))):
            if row >= n_tokens:
                dropped += max(0, int(new[r])) - i
                break
            p = n + i
            if not full and (p >= width * BLOCK or (p % BLOCK == 0 and not free)):
                full = True
            if full:
                dropped += 1
                row += 1
                continue
            if p % BLOCK == 0:
                table[r, p // BLOCK] = free.pop()
            b = table[r, p // BLOCK]
            slots[row] = b * BLOCK + p % BLOCK
            positions[row] = p
            end = p + 1
            if runs and runs[-1][2] == r and runs[-1][3] // BLOCK == p // BLOCK:
                runs[-1][1] += 1
            else:
                runs.append([row, 1, r, p])
            row += 1
        ends[r] = end
    room = min(n_tokens, (n_tokens + 126 * min(n_tokens, R)) // BLOCK)
    assert len(runs) <= room
    chunks = np.zeros((room, 4), dtype=np.int64)
    if runs:
        chunks[:len(runs)] = runs
    return table, slots, positions, chunks, ends, np.array([len(free), min(dropped, 2**31 - 1)])


def tables(lens, width, n_blocks, rng):
    """Random tables of requests with `lens` tokens, and the free list."""
    order = rng.permutation(n_blocks)
    table, at = np.full((len(lens), width), -1, dtype=np.int64), 0
    for r, n in enumerate(lens):
        b = -(-int(n) // BLOCK)
        table[r, :b] = order[at:at + b]
        at += b
    free = np.zeros(n_blocks, dtype=np.int64)
    free[:n_blocks - at] = order[at:]
    return table, free, np.array([n_blocks - at, 0])


def rope(x, cos, sin):
    """Pairs of x (..., D) turned, products and sums rounded in fp32."""
    a, b = x[..., 0::2], x[..., 1::2]
    out = np.empty_like(x)
    out[..., 0::2] = a * cos - b * sin
    out[..., 1::2] = b * cos + a * sin
    return out


def codes(x, scale):
    """int8 codes of x at a scale, steps rounded in fp32."""
    if not (scale > 0 and np.isfinite(scale)):
        return np.zeros(x.shape, dtype=np.int8)
    return np.clip(np.rint(x / scale), -127, 127).astype(np.int8)


def append(qkv, slots, positions, chunks, cos, sin, k, v, ks, vs, H):
    """Chunk by chunk in fp32; the cache arrays are updated.  Returns q in
    64 bits (NaN rows where nothing is written)."""
    n_blocks, Hk, _, D = k.shape
    qkv = qkv.astype(np.float32)
    n = qkv.shape[0]
    q = np.full((n, H, D), np.nan)
    for row0, count, _, _ in chunks:
        if count == 0:
            continue
        rows = slice(row0, row0 + count)
        block, before = slots[row0] // BLOCK, slots[row0] % BLOCK
        c, s = cos[positions[rows]][:, None], sin[positions[rows]][:, None]
        x = qkv[rows].reshape(count, H + 2 * Hk, D)
        q[rows] = rope(x[:, :H].astype(np.float64), c.astype(np.float64),
                       s.astype(np.float64)) / math.sqrt(D)
        keys, values = rope(x[:, H:H + Hk], c, s), x[:, H + Hk:]
        for h in range(Hk):
            for new, cache, scale in ((keys[:, h], k[block, h], ks), (values[:, h], v[block, h].T, vs)):
                old = np.float32(scale[block, h]) if before else np.float32(0)
                m = np.abs(new)
                top = np.float32(np.where(np.isnan(m), np.inf, m).max())
                grown = np.maximum(old, top * (np.float32(1) / np.float32(127)))
                if before and grown > old:
                    cache[:before] = codes(cache[:before].astype(np.float32) * old, grown)
                cache[before:before + count] = codes(new, grown)
                scale[block, h] = grown
    return q


def attention(q, chunks, table, k, v, ks, vs, lens, softcap=0.0, window=0, slopes=None,
              prefix=None):
    """(out, bound): 64 bits, and per element what fp32 arithmetic with 24-bit
    (out: fp32) factors may lose, see the terms below; rows without a chunk are
    NaN."""
    n_blocks, Hk, _, D = k.shape
    n, H = q.shape[0], q.shape[1] // D
    G = H // Hk
    out = np.full((n, H, D), np.nan)
    score_loss = np.zeros((n, H))     # in units of the rounding step
    top = np.zeros((n, H))
    for row0, count, r, pos0 in chunks:
        for t in range(row0, row0 + count):
            i = pos0 + t - row0
            pre = min(max(int(prefix[r]), 0), int(lens[r])) if prefix is not None else 0
            ids = table[r, :-(-max(i + 1, pre) // BLOCK)]
            good = np.repeat((ids >= 0) & (ids < n_blocks), BLOCK)
            ids = np.clip(ids, 0, n_blocks - 1)
            j = np.arange(len(ids) * BLOCK)
            seen = j <= i
            if window:
                seen &= j > i - window
            seen = (seen | (j < pre)) & good
            for h in range(H):
                g = h // G
                out[t, h] = 0
                if not seen.any():
                    continue
                keys = (k[ids, g].astype(np.float64) * ks[ids, g][:, None, None]).reshape(-1, D)[seen]
                values = (v[ids, g].astype(np.float64) * vs[ids, g][:, None, None]) \
                    .transpose(0, 2, 1).reshape(-1, D)[seen]
                x = q[t, h * D:(h + 1) * D].astype(np.float64)
                s = keys @ x
                size = np.abs(keys) @ np.abs(x) + np.abs(keys).sum(1) * np.abs(x).max()
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                    size = size + 8 * softcap
                if slopes is not None:
                    s = s + slopes[h] * (j[seen] - i)
                    size = size + 2 * np.abs(slopes[h] * (j[seen] - i))
                w = np.exp(s - s.max())
                out[t, h] = w @ values / w.sum()
                score_loss[t, h] = (size + np.abs(s)).max()
                top[t, h] = np.abs(values).max()
    return out, score_loss, top


def rules(logits, history=None, lens=None, prompt=None, repetition=None, frequency=None,
          presence=None, ids=None, bias=None, mask=None):
    """Token by token in fp32: (logits, tokens)."""
    f = np.float32
    x = logits.astype(f).copy()
    B, V = x.shape
    tokens = np.full(B, -1)
    with np.errstate(all="ignore"):
        for b in range(B):
            if history is not None:
                seq = [int(t) for t in history[b, :max(0, min(int(lens[b]), history.shape[1]))]]
                at = int(prompt[b]) if prompt is not None else 0
                for t in set(seq):
                    if not 0 <= t < V:
                        continue
                    if repetition is not None:
                        r = f(repetition[b])
                        x[b, t] = x[b, t] / r if x[b, t] > 0 else x[b, t] * r
                    n = sum(1 for i, s in enumerate(seq) if s == t and i >= at)
                    if n:
                        x[b, t] = x[b, t] - (f(frequency[b]) * f(n) if frequency is not None else f(0))
                        x[b, t] = x[b, t] - (f(presence[b]) if presence is not None else f(0))
            if ids is not None:
                for t, value in {int(t): value for t, value in zip(ids[b], bias[b])}.items():
                    if 0 <= t < V:
                        x[b, t] = x[b, t] + f(value)
            if mask is not None:
                for t in range(V):
                    if not int(mask[b, t // 32]) >> (t % 32) & 1:
                        x[b, t] = -np.inf
            best = -np.inf
            for t in range(V):
                if x[b, t] > best:
                    best, tokens[b] = x[b, t], t
    return x, tokens
