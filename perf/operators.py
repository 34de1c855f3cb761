"""The operators that serve requests of different lengths from one 8-bit key /
value cache, as cases that can be timed.

A case is a dict of plain values; its ``kind`` names the operator:

* ``plan``: block tables, slot maps, positions and the list of work chunks of
  one serving step from the requests' lengths, on the GPU;
* ``append``: RoPE of the queries and keys of a step's tokens and the append
  of keys and values to the cache (int8 codes, one fp32 scale for each block
  of 64 tokens and head), then the touched tokens read back;
* ``attention``: attention of the step's queries over the cached blocks, with
  scores that may be capped, biased by distance, windowed or have a
  bidirectional prefix;
* ``logits``: penalties for repeated tokens, biases and grammar masks on the
  logits, and the greedy choice.

Sizes: the 2.2B shape's 20 heads of 128, context 1024 and vocabularies of
32000 and 50257, and generic ones around them (grouped heads, head dims from
64 to 256, caches of tens of thousands of tokens).
"""
import math

import torch

own = False

BLOCK = 64          # tokens of a cache block
HEADS, HEAD_DIM = 20, 128
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # a decode step of a small server: one new token for each request
        _plan("plan, 8 requests decode", 8, 1024, 8, "decode"),
        # a large mixed step: prompts and single tokens of many requests
        _plan("plan, 700 requests mixed", 700, 8192, 30011, "mixed"),
        # one token of a few requests through a layer, module numerics (fp32)
        _append("append, 5 tokens", 5, 5, 900, HEADS, HEADS, HEAD_DIM, "float32"),
        # a decode batch with grouped heads, bf16 activations
        _append("append, 96 tokens grouped", 96, 96, 4000, 32, 8, 128, "bfloat16"),
        # ragged prompts of the 2.2B shape: the largest append
        _append("append, 6001 prompt tokens", 9, 6001, 500, HEADS, HEADS, HEAD_DIM, "float32"),
        # the smallest attention: one token of three requests, short caches
        _attention("attention, 3 requests decode", 3, 3, 200, HEADS, HEADS, HEAD_DIM, "float32"),
        # a decode batch of the 2.2B shape with its full context
        _attention("attention, 64 requests decode", 64, 64, 960, HEADS, HEADS, HEAD_DIM, "bfloat16"),
        # few requests far into long documents, grouped heads: the longest cache
        _attention("attention, 6 requests of 40000", 6, 6, 40000, 32, 8, 128, "bfloat16"),
        # ragged prompts of the 2.2B shape at once, module numerics: the largest
        _attention("attention, 8003 prompt tokens", 2, 8003, 0, HEADS, HEADS, HEAD_DIM, "float32"),
        # prompt chunks in the middle of requests with capped scores, distance
        # biases, a window and prefixes
        _attention("attention, 1500 tokens with every rule", 4, 1500, 3000, 24, 8, 64, "bfloat16",
                   softcap=30.0, window=1000, slopes=True, prefix=True),
        # the tied head's logits of one request
        _logits("logits, 1 of 50257", 1, 50257, 700, "float32"),
        # a full batch over a large vocabulary with long histories
        _logits("logits, 160 of 131077", 160, 131077, 4000, "float32"),
    ]


def _plan(name, requests, most, tokens, mode):
    return {"name": name, "kind": "plan", "requests": requests, "most": most, "tokens": tokens,
            "mode": mode}


def _append(name, requests, tokens, past, heads, kv_heads, head_dim, dtype):
    return {"name": name, "kind": "append", "requests": requests, "tokens": tokens, "past": past,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype}


def _attention(name, requests, tokens, past, heads, kv_heads, head_dim, dtype, softcap=0.0,
               window=0, slopes=False, prefix=False):
    return {"name": name, "kind": "attention", "requests": requests, "tokens": tokens,
            "past": past, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype, "softcap": softcap, "window": window, "slopes": slopes,
            "prefix": prefix}


def _logits(name, rows, vocab, history, dtype):
    return {"name": name, "kind": "logits", "rows": rows, "vocab": vocab, "history": history,
            "dtype": dtype}


def _spread(rng, low, high):
    """A whole number, spread evenly over the range's logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "append", "attention", "attention", "attention", "logits"])
    dtype = rng.choice(sorted(DTYPES))
    if kind == "plan":
        requests = _spread(rng, 1, 700)
        if rng.random() < 0.5:
            case = _plan("", requests, _spread(rng, 64, 8192), requests, "decode")
        else:
            case = _plan("", requests, _spread(rng, 512, 8192),
                         _spread(rng, requests, 30000), "mixed")
    elif kind == "logits":
        vocab = _spread(rng, 1000, 131077)
        case = _logits("", _spread(rng, 1, 160), vocab, _spread(rng, 1, 4000), dtype)
    else:
        kv_heads = rng.choice([1, 2, 4, 5, 8, 12, 20])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8] if kv_heads <= 5 else [1, 1, 2, 3])
        head_dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        decode = rng.random() < 0.5
        if kind == "append":
            # no more values than the largest listed append reads
            most = max(1, 6001 * 3 * HEADS * HEAD_DIM // ((heads + 2 * kv_heads) * head_dim))
            requests = _spread(rng, 1, 96 if decode else 9)
            tokens = requests if decode else _spread(rng, requests, max(requests, min(6001, most)))
            case = _append("", requests, tokens, _spread(rng, 1, 4000 if decode else 500), heads,
                           kv_heads, head_dim, dtype)
        else:
            rules = {"softcap": rng.choice([0.0, 0.0, 20.0, 50.0]),
                     "window": rng.choice([0, 0, _spread(rng, 1, 2000)]),
                     "slopes": rng.random() < 0.3, "prefix": rng.random() < 0.3}
            # no more cached values and no more products than the largest
            # listed cases
            if decode:
                tokens = requests = _spread(rng, 1, 64)
                values = 6 * 40000 * 8 * 128
                past = _spread(rng, 1, max(1, min(40000, values // (requests * kv_heads * head_dim))))
            else:
                requests = rng.randint(1, 4)
                past = rng.choice([0, _spread(rng, 1, 3000)])
                tokens = _spread(rng, requests, 8003)
                while tokens * (past + tokens / requests / 2) * heads * head_dim > \
                        8003 * 2000 * HEADS * HEAD_DIM:
                    tokens = max(requests, tokens * 3 // 4)
            case = _attention("", requests, tokens, past, heads, kv_heads, head_dim, dtype, **rules)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    return {"plan": _prepare_plan, "append": _prepare_append, "attention": _prepare_attention,
            "logits": _prepare_logits}[case["kind"]](case, seed)


def _host(seed):
    return torch.Generator().manual_seed(int(seed))


def _split(total, parts, g):
    """total as `parts` whole numbers of at least one each (total >= parts)."""
    if parts == 1:
        return torch.tensor([total])
    cuts = torch.randperm(total - 1, generator=g)[:parts - 1].sort().values + 1
    edges = torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([total])])
    return edges[1:] - edges[:-1]


def _blocks(tokens):
    return (tokens + BLOCK - 1) // BLOCK


def _tables(lens, width, n_blocks, g):
    """Block tables (-1 past each request's blocks) over blocks in random
    order, and the blocks left over."""
    need = _blocks(lens)
    order = torch.randperm(n_blocks, generator=g)
    used = int(need.sum())
    table = torch.full((lens.numel(), width), -1, dtype=torch.int64)
    inside = torch.arange(width) < need[:, None]
    table[inside] = order[:used]
    return table.int(), order[used:].int()


def _prepare_plan(case, seed):
    g = _host(seed)
    R, most, tokens = case["requests"], case["most"], case["tokens"]
    width = _blocks(most)
    if case["mode"] == "decode":
        lens = torch.randint(0, most, (R,), generator=g)
        new = (torch.rand(R, generator=g) < 0.97).long()   # a few requests wait
    else:
        # a third of the requests start with a prompt, the others add a token
        lens = torch.randint(0, max(1, most // 2), (R,), generator=g)
        new = torch.ones(R, dtype=torch.int64)
        starts = torch.rand(R, generator=g) < 0.34
        starts[0] = True
        share = max(0, tokens - R) // int(starts.sum())
        longest = max(2, min(2 * share, most // 2))
        new[starts] = torch.randint(1, longest + 1, (int(starts.sum()),), generator=g)
        lens[starts] = 0
        new = torch.minimum(new, (tokens - (new.cumsum(0) - new)).clamp(min=0))
    n_blocks = int(_blocks(lens + new).sum()) + 37
    table, rest = _tables(lens, width, n_blocks, g)
    free = torch.zeros(n_blocks, dtype=torch.int32)
    free[:rest.numel()] = rest
    dev = "cuda"
    return {"case": case, "table": table.to(dev), "lens": lens.int().to(dev),
            "new": new.int().to(dev), "free": free.to(dev), "tokens": tokens,
            "state": torch.tensor([rest.numel(), 0], dtype=torch.int32, device=dev)}


def _step(case, g, n_extra=11):
    """Lengths, tables and the plan's slots, positions and chunks of a step:
    every request has about `past` tokens cached and gets its share of the new
    ones."""
    R, past = case["requests"], case["past"]
    lens = torch.randint((past + 1) // 2, past + 1, (R,), generator=g)
    lens[0] = past
    new = _split(case["tokens"], R, g)
    ends = lens + new
    width = int(_blocks(ends).max())
    n_blocks = int(_blocks(ends).sum()) + n_extra
    table, _ = _tables(ends, width, n_blocks, g)
    r = torch.repeat_interleave(torch.arange(R), new)
    first = new.cumsum(0) - new
    pos = lens[r] + torch.arange(case["tokens"]) - first[r]
    slots = table.long()[r, pos // BLOCK] * BLOCK + pos % BLOCK
    count = (ends - 1) // BLOCK - lens // BLOCK + 1
    cr = torch.repeat_interleave(torch.arange(R), count)
    j = torch.arange(int(count.sum())) - (count.cumsum(0) - count)[cr]
    begin = torch.maximum(lens[cr], (lens[cr] // BLOCK + j) * BLOCK)
    end = torch.minimum(ends[cr], (lens[cr] // BLOCK + j + 1) * BLOCK)
    chunks = torch.stack([first[cr] + begin - lens[cr], end - begin, cr, begin], dim=1)
    dev = "cuda"
    return {"lens": lens, "new": new, "ends": ends, "n_blocks": n_blocks, "width": width,
            "table": table.to(dev), "slots": slots.int().to(dev), "positions": pos.int().to(dev),
            "chunks": chunks.int().to(dev).contiguous(), "ends_dev": ends.int().to(dev),
            "request": r.to(dev)}


def _cache(n_blocks, kv_heads, head_dim, gen, dev):
    """Codes as quantized N(0, 1) keys and values leave them, and scales of
    blocks of different size."""
    def codes(*shape):
        return torch.randn(*shape, generator=gen, device=dev).mul_(127 / 3.6).round_() \
            .clamp_(-127, 127).to(torch.int8)
    k = codes(n_blocks, kv_heads, BLOCK, head_dim)
    v = codes(n_blocks, kv_heads, head_dim, BLOCK)
    ks = torch.rand(n_blocks, kv_heads, generator=gen, device=dev) * 0.02 + 0.02
    vs = torch.rand(n_blocks, kv_heads, generator=gen, device=dev) * 0.02 + 0.02
    return k, v, ks, vs


def _prepare_append(case, seed):
    s = _step(case, _host(seed))
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(int(seed) + 1)
    H, Hk, D = case["heads"], case["kv_heads"], case["head_dim"]
    k, v, ks, vs = _cache(s["n_blocks"], Hk, D, gen, dev)
    qkv = torch.randn(case["tokens"], (H + 2 * Hk) * D, generator=gen, device=dev)
    most = int(s["ends"].max())
    inv = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    angles = torch.arange(most, dtype=torch.float64)[:, None] * inv
    # what the step touches: the tokens before each request's first new one in
    # its block (-1 in the place of those that are not there), and the new ones
    lens = s["lens"].to(dev)
    block = s["table"].long()[torch.arange(case["requests"], device=dev), lens // BLOCK]
    i = torch.arange(BLOCK, device=dev)
    before = torch.where(i < (lens % BLOCK)[:, None], block[:, None] * BLOCK + i, -1)
    read = torch.cat([before.flatten().int(), s["slots"]])
    s.update(case=case, qkv=qkv.to(DTYPES[case["dtype"]]), k=k, v=v, ks=ks, vs=vs,
             cos=angles.cos().float().to(dev), sin=angles.sin().float().to(dev),
             read=read)
    return s


def _prepare_attention(case, seed):
    s = _step(case, _host(seed))
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(int(seed) + 1)
    g = _host(seed + 2)
    H, Hk, D = case["heads"], case["kv_heads"], case["head_dim"]
    k, v, ks, vs = _cache(s["n_blocks"], Hk, D, gen, dev)
    # scaled queries, rows of different sharpness
    q = torch.randn(case["tokens"], H * D, generator=gen, device=dev) * D ** -0.5
    q = q * (torch.rand(case["tokens"], 1, generator=gen, device=dev) * 2.5 + 0.5)
    slopes = (2.0 ** (-8.0 * torch.arange(1, H + 1) / H)).float().to(dev) if case["slopes"] else None
    prefix = None
    if case["prefix"]:
        prefix = (torch.rand(case["requests"], generator=g) * s["ends"]).int().to(dev)
    s.update(case=case, q=q.to(DTYPES[case["dtype"]]), k=k, v=v, ks=ks, vs=vs, slopes=slopes,
             prefix=prefix)
    return s


def _prepare_logits(case, seed):
    g = _host(seed)
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(int(seed) + 1)
    B, V, most = case["rows"], case["vocab"], case["history"]
    logits = torch.randn(B, V, generator=gen, device=dev) * 4
    logits = (30 * torch.tanh(logits / 30)).to(DTYPES[case["dtype"]])
    # text repeats itself: histories of few different tokens, the likely ones
    # among them
    top = logits.float().topk(min(V, 64), dim=1).indices
    history = torch.randint(0, V, (B, most), generator=gen, device=dev)
    pick = torch.randint(0, top.shape[1], (B, most), generator=gen, device=dev)
    often = torch.rand(B, most, generator=gen, device=dev) < 0.2
    history = torch.where(often, top.gather(1, pick), history).int()
    lens = torch.randint((most + 1) // 2, most + 1, (B,), generator=g)
    prompt = (lens * torch.rand(B, generator=g)).long()
    ids = torch.randint(0, V, (B, 40), generator=g)
    bias = torch.randn(B, 40, generator=g) * 2
    bias[:, ::7] = -100.0   # banned tokens
    # grammar masks: most rows allow about half the vocabulary, one nothing
    words = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), generator=gen, device=dev,
                          dtype=torch.int64).int()
    words[::3] = -1
    if B > 4:
        words[4] = 0
    return {"case": case, "logits": logits, "history": history, "lens": lens.int().to(dev),
            "prompt": prompt.int().to(dev),
            "repetition": (1 + 0.3 * torch.rand(B, generator=g)).to(dev),
            "frequency": (0.4 * torch.rand(B, generator=g)).to(dev),
            "presence": (0.5 * torch.rand(B, generator=g)).to(dev),
            "ids": ids.int().to(dev), "bias": bias.to(dev), "mask": words}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return {"plan": _run_plan, "append": _run_append, "attention": _run_attention,
            "logits": _run_logits}[state["case"]["kind"]](state)


def _run_plan(s):
    if own:
        from nativebit_amd import ops
        p = ops.kv_plan(s["table"], s["lens"], s["new"], s["free"], s["state"], s["tokens"])
        return {"table": s["table"], "slots": p.slots, "positions": p.positions,
                "chunks": p.chunks, "lens": p.lens, "state": p.state}
    table, n = s["table"], s["tokens"]
    R, width = table.shape
    n_blocks = s["free"].numel()
    dev = table.device
    lens = s["lens"].long().clamp(0, width * BLOCK)
    asked = s["new"].long().clamp(min=0)
    new = torch.minimum(asked, (n - (asked.cumsum(0) - asked)).clamp(min=0))
    last = new.cumsum(0)
    first = last - new
    ends = (lens + new).clamp(max=width * BLOCK)
    have = _blocks(lens)
    need = _blocks(ends) - have
    base = need.cumsum(0) - need
    left = s["state"][0].long().clamp(0, n_blocks)
    got = torch.minimum(need, (left - base).clamp(min=0))
    ends = torch.minimum(ends, (have + got) * BLOCK)
    # the new blocks from the end of the free list, requests in order
    j = torch.arange(width, device=dev)
    fresh = (j >= have[:, None]) & (j < (have + got)[:, None])
    rank = base[:, None] + j - have[:, None]
    ids = s["free"][(left - 1 - rank).clamp(0, n_blocks - 1)]
    table.copy_(torch.where(fresh, ids, table))
    # slots and positions of the step's rows
    t = torch.arange(n, device=dev)
    r = torch.searchsorted(last, t, right=True).clamp(max=R - 1)
    pos = lens[r] + t - first[r]
    stored = (t < last[-1]) & (pos < ends[r])
    pos = torch.where(stored, pos, 0)
    block = table[r, pos // BLOCK].long()
    good = stored & (block >= 0) & (block < n_blocks)
    slots = torch.where(good, block * BLOCK + pos % BLOCK, -1)
    # runs of rows of one request within one block
    most = _chunks_bound(n, R)
    count = torch.where(ends > lens, (ends - 1) // BLOCK - lens // BLOCK + 1, 0)
    upto = count.cumsum(0)
    i = torch.arange(most, device=dev)
    cr = torch.searchsorted(upto, i, right=True).clamp(max=R - 1)
    b = lens[cr] // BLOCK + i - (upto - count)[cr]
    begin = torch.maximum(lens[cr], b * BLOCK)
    end = torch.minimum(ends[cr], (b + 1) * BLOCK)
    chunks = torch.stack([first[cr] + begin - lens[cr], end - begin, cr, begin], dim=1)
    chunks = torch.where((i < upto[-1])[:, None], chunks, 0)
    state = torch.stack([left - got.sum(), asked.sum() - (ends - lens).sum()])
    return {"table": table, "slots": slots.int(), "positions": pos.int(), "chunks": chunks.int(),
            "lens": ends.int(), "state": state.int()}


def _chunks_bound(tokens, requests):
    """The most chunks that `tokens` rows of `requests` requests make."""
    return min(tokens, (tokens + 126 * min(tokens, requests)) // BLOCK)


def _kv_plan(s):
    from nativebit_amd import ops
    return ops.KVPlan(s["slots"], s["positions"], s["chunks"], s["ends_dev"], None)


def _run_append(s):
    case = s["case"]
    H, Hk, D = case["heads"], case["kv_heads"], case["head_dim"]
    if own:
        from nativebit_amd import ops
        q = ops.kv8_append(s["qkv"], _kv_plan(s), s["cos"], s["sin"], s["k"], s["v"], s["ks"],
                           s["vs"], H)
        keys, values = ops.kv8_read(s["read"], s["k"], s["v"], s["ks"], s["vs"])
        return {"q": q, "keys": keys, "values": values}
    n = case["tokens"]
    pos, slots, c = s["positions"].long(), s["slots"].long(), s["chunks"].long()
    rows = s["qkv"].float().view(n, H + 2 * Hk, D)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turn(x):
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)

    q = turn(rows[:, :H]) * D ** -0.5
    new_k, new_v = turn(rows[:, H:H + Hk]), rows[:, H + Hk:]
    block, inside = slots // BLOCK, slots % BLOCK
    chunk = torch.searchsorted(c[:, 0].contiguous(), torch.arange(n, device=pos.device),
                               right=True) - 1
    touched, before = block[c[:, 0]], inside[c[:, 0]]
    held = torch.arange(BLOCK, device=pos.device) < before[:, None]   # (chunk, token)

    def scales(scale, x):
        most = torch.zeros(c.shape[0], Hk, device=x.device).scatter_reduce(
            0, chunk[:, None].expand(n, Hk), x.abs().amax(-1), "amax")
        old = torch.where((before > 0)[:, None], scale[touched], 0.0)
        return old, torch.maximum(old, most / 127)

    def code(x, scale):
        return torch.where(scale > 0, x / scale, 0.0).round().clamp(-127, 127).to(torch.int8)

    old, new = scales(s["ks"], new_k)
    codes = s["k"][touched]
    again = code(codes.float() * old[:, :, None, None], new[:, :, None, None])
    s["k"][touched] = torch.where(held[:, None, :, None], again, codes)
    s["k"][block, :, inside] = code(new_k, new[chunk][:, :, None])
    s["ks"][touched] = new
    old, new = scales(s["vs"], new_v)
    codes = s["v"][touched]
    again = code(codes.float() * old[:, :, None, None], new[:, :, None, None])
    s["v"][touched] = torch.where(held[:, None, None, :], again, codes)
    s["v"][block, :, :, inside] = code(new_v, new[chunk][:, :, None])
    s["vs"][touched] = new
    at = s["read"].long().clamp(min=0)
    block, inside = at // BLOCK, at % BLOCK
    none = (s["read"] < 0)[:, None, None]
    keys = s["k"][block, :, inside].float() * s["ks"][block][:, :, None]
    values = s["v"][block, :, :, inside].float() * s["vs"][block][:, :, None]
    return {"q": q.reshape(n, H * D).to(s["qkv"].dtype), "keys": keys.masked_fill(none, 0.0),
            "values": values.masked_fill(none, 0.0)}


def _run_attention(s):
    case = s["case"]
    if own:
        from nativebit_amd import ops
        return ops.kv8_attention(s["q"], _kv_plan(s), s["table"], s["k"], s["v"], s["ks"], s["vs"],
                                 softcap=case["softcap"], window=case["window"],
                                 slopes=s["slopes"], prefix=s["prefix"])
    n, H, Hk, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    R, width = s["table"].shape
    S, T, G = width * BLOCK, int(s["new"].max()), H // Hk
    dev = s["q"].device
    at = s["table"].long().clamp(min=0)
    keys = (s["k"][at].float() * s["ks"][at][..., None, None]).transpose(1, 2).reshape(R, Hk, S, D)
    values = (s["v"][at].float() * s["vs"][at][..., None, None]).transpose(1, 2) \
        .transpose(3, 4).reshape(R, Hk, S, D)
    # the rows of each request, padded to the longest
    r = s["request"]
    first = (s["new"].cumsum(0) - s["new"]).to(dev)
    inside = torch.arange(n, device=dev) - first[r]
    q = torch.zeros(R, T, H, D, device=dev)
    q[r, inside] = s["q"].float().view(n, H, D)
    q = q.view(R, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(R, Hk, G * T, D)
    scores = torch.matmul(q, keys.transpose(2, 3)).view(R, Hk, G, T, S)
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    i = s["lens"].to(dev)[:, None, None] + torch.arange(T, device=dev)[:, None]   # (R, T, 1)
    j = torch.arange(S, device=dev)
    if s["slopes"] is not None:
        scores = scores + s["slopes"].view(Hk, G, 1, 1) * (j - i).float()[:, None, None]
    seen = j <= i
    if case["window"]:
        seen = seen & (j > i - case["window"])
    if s["prefix"] is not None:
        seen = seen | (j < torch.minimum(s["prefix"], s["ends_dev"])[:, None, None])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul((e / e.sum(-1, keepdim=True)).view(R, Hk, G * T, S), values)
    out = out.view(R, Hk, G, T, D).permute(0, 3, 1, 2, 4).reshape(R, T, H * D)
    return out[r, inside].to(s["q"].dtype)


def _run_logits(s):
    if own:
        from nativebit_amd import ops
        out, tokens = ops.logits_rules(
            s["logits"], history=s["history"], lens=s["lens"], prompt_lens=s["prompt"],
            repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
            bias_ids=s["ids"], bias=s["bias"], mask=s["mask"], choose=True)
        return {"logits": out, "tokens": tokens}
    x = s["logits"].float()
    B, V = x.shape
    at = torch.arange(s["history"].shape[1], device=x.device)
    ids = s["history"].long()
    held = (at < s["lens"][:, None]).float()
    answer = held * (at >= s["prompt"][:, None])
    seen = torch.zeros_like(x).scatter_add_(1, ids, held) > 0
    count = torch.zeros_like(x).scatter_add_(1, ids, answer)
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count
    x = x - s["presence"][:, None] * (count > 0)
    # an id listed twice has its last value
    ids = s["ids"].long()
    order = torch.arange(ids.shape[1], device=x.device).expand(B, -1)
    last = torch.full((B, V), -1, device=x.device).scatter_reduce_(1, ids, order, "amax")
    x = x + torch.where(last >= 0, s["bias"].gather(1, last.clamp(min=0)), 0.0)
    v = torch.arange(V, device=x.device)
    x = x.masked_fill((s["mask"][:, v // 32] >> (v % 32).int()) & 1 == 0, -math.inf)
    best = x.amax(1, keepdim=True)
    tokens = torch.where(x == best, v, V).amin(1)
    return {"logits": x, "tokens": torch.where(best[:, 0] > -math.inf, tokens, -1).int()}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "plan":
        R, n = case["requests"], case["tokens"]
        # lengths and counts in and out, slots, positions, chunks, new blocks
        return {"bytes": 4.0 * (4 * R + 2 * n + 4 * _chunks_bound(n, R) + 2 * n / BLOCK),
                "flops": 0.0}
    if kind == "logits":
        B, V = case["rows"], case["vocab"]
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": B * (V * (size + 4 + 1 / 8) + 3.0 * case["history"]), "flops": 8.0 * B * V}
    n, H, Hk, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    R, past = case["requests"], case["past"]
    size = 2 if case["dtype"] == "bfloat16" else 4
    cached = R * 0.75 * past if R > 1 else past    # tokens before the step
    if kind == "append":
        # rows, codes and angles of the step; then its codes and about half a
        # block of earlier ones for each request read back, fp32 rows written
        return {"bytes": n * D * (size * (2 * H + 2 * Hk) + 2.0 * Hk + 4) +
                Hk * D * ((n + 32.0 * R) * 2 + (n + 64.0 * R) * 8), "flops": n * D * (3.0 * H + 6.0 * Hk)}
    tokens = cached + n
    share = n / R
    seen = 0.75 * past + share / 2 if R > 1 else past + share / 2
    if case["window"] and not case["prefix"]:
        seen = min(seen, case["window"])
        tokens = min(tokens, R * (case["window"] + share))
    return {"bytes": tokens * Hk * (2 * D + 8 / BLOCK) + 2.0 * n * H * D * size,
            "flops": 4.0 * n * seen * H * D}


# ---------------------------------------------------------------------------
# the same from the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None
    s = prepare(case, seed)
    if kind == "logits":
        return {"logits": _exact_logits(s), "tokens": None}
    H, D = case["heads"], case["head_dim"]
    if kind == "append":
        n = case["tokens"]
        z = torch.view_as_complex(s["qkv"][:, :H * D].double().view(n, H, D // 2, 2).contiguous())
        at = s["positions"].long()
        w = torch.complex(s["cos"].double()[at], s["sin"].double()[at])[:, None]
        # (what is held in 8 bits follows from roundings, which 64 bits decide otherwise)
        return {"q": torch.view_as_real(z * w).reshape(n, H * D) / math.sqrt(D),
                "keys": None, "values": None}
    return _exact_attention(s, case)


def _exact_logits(s):
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    hist, lens, prompt = (s[k].cpu().numpy() for k in ("history", "lens", "prompt"))
    rep, freq, pres, bias = (s[k].double().cpu().numpy()
                             for k in ("repetition", "frequency", "presence", "bias"))
    ids = s["ids"].cpu().numpy()
    bits = np.unpackbits(s["mask"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")
    for b in range(x.shape[0]):
        for v in np.unique(hist[b, :lens[b]]):
            x[b, v] = x[b, v] / rep[b] if x[b, v] > 0 else x[b, v] * rep[b]
        tokens, counts = np.unique(hist[b, prompt[b]:lens[b]], return_counts=True)
        x[b, tokens] -= freq[b] * counts + pres[b]
        for v, value in dict(zip(ids[b].tolist(), bias[b].tolist())).items():
            x[b, v] += value
        x[b, bits[b, :x.shape[1]] == 0] = -np.inf
    return x


def _exact_attention(s, case):
    """Request by request and head by head."""
    H, Hk, D = case["heads"], case["kv_heads"], case["head_dim"]
    lens, new = s["lens"].tolist(), s["new"].tolist()
    out = torch.zeros(case["tokens"], H, D, dtype=torch.float64, device=s["q"].device)
    row = 0
    for r, (before, count) in enumerate(zip(lens, new)):
        end = before + count
        ids = s["table"][r, :-(-end // BLOCK)].long()
        i = torch.arange(before, end, device=out.device)[:, None]
        j = torch.arange(end, device=out.device)[None]
        seen = j <= i
        if case["window"]:
            seen &= i - j < case["window"]
        if s["prefix"] is not None:
            seen |= j < s["prefix"][r]
        q = s["q"][row:row + count].double().view(count, H, D)
        for h in range(H):
            g = h // (H // Hk)
            k = (s["k"][ids, g].double() * s["ks"][ids, g].double()[:, None, None]).reshape(-1, D)
            v = s["v"][ids, g].double() * s["vs"][ids, g].double()[:, None, None]
            v = v.permute(0, 2, 1).reshape(-1, D)
            x = q[:, h] @ k[:end].T
            if case["softcap"]:
                x = case["softcap"] * (x / case["softcap"]).tanh()
            if s["slopes"] is not None:
                x = x - s["slopes"][h].double() * (i - j)
            x = x.masked_fill(~seen, -math.inf)
            out[row:row + count, h] = torch.softmax(x, dim=1) @ v[:end]
        row += count
    return out.view(case["tokens"], H * D)
