"""The operators of a decoding step in 8 bits with a drawn token at its end, as
cases that can be timed.

A case is a dict of plain values; its ``kind`` names the operator:

* ``norm``: the residual's addition and the root-mean-square norm, the rows in
  8 bits with one scale each;
* ``quantize``: rows in 8 bits with one scale each;
* ``linear``: rows in 8 bits times packed 3-bit weights whose codebooks are in
  8 bits, with bias, activation and residual in the epilogue;
* ``sample``: tokens drawn from logits with temperature, top-k, top-p and min-p
  by given random numbers, and their log-probabilities.

Sizes: the 2.2B shape (2560 wide, 6912 hidden, blocks of 128 weights with 8
entries), its vocabulary of 50257, and generic ones around them.
"""
import math

import torch

own = False

WIDTH, HIDDEN, BLOCK, ENTRIES = 2560, 6912, 128, 8
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # the norm of one decoded token: latency
        _norm("norm, 1 row", 1, WIDTH, "float32", False),
        # a block's second norm over a long prompt, module numerics
        _norm("norm + residual, 2048 rows", 2048, WIDTH, "float32", True),
        # the gated products of a small decode batch, for the down projection
        _quantize("quantize, 8 rows", 8, HIDDEN, "bfloat16"),
        # the same of a long prompt
        _quantize("quantize, 2048 rows", 2048, HIDDEN, "float32"),
        # the output projection of one decoded token, added to the stream
        _linear("linear, 1 row + residual", 1, WIDTH, WIDTH, "float32", residual=True),
        # q|k|v of a decode batch
        _linear("linear, 9 rows", 9, 3 * WIDTH, WIDTH, "float32"),
        # the down projection of a short ragged batch, added to the stream
        _linear("linear, 129 rows + residual", 129, WIDTH, HIDDEN, "float32", residual=True),
        # an odd layer with a bias and an activation, generic
        _linear("linear, 500 rows bias gelu", 500, 5003, 1280, "bfloat16", bias=True,
                activation="gelu"),
        # gate|up of a long prompt with the gated product: the largest
        _linear("linear, 2048 rows swiglu", 2048, 2 * HIDDEN, WIDTH, "bfloat16",
                activation="swiglu"),
        # one request, temperature and nucleus
        _sample("sample, 1 of 50257", 1, 50257, "float32", top_p=True),
        # a decode batch of the model dtype's logits, every rule
        _sample("sample, 48 of 50257 every rule", 48, 50257, "bfloat16", top_k=True, top_p=True,
                min_p=True),
        # a full batch over a large vocabulary, every rule
        _sample("sample, 160 of 131077 every rule", 160, 131077, "float32", top_k=True,
                top_p=True, min_p=True),
    ]


def _norm(name, rows, width, dtype, residual):
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "dtype": dtype,
            "residual": residual}


def _quantize(name, rows, width, dtype):
    return {"name": name, "kind": "quantize", "rows": rows, "width": width, "dtype": dtype}


def _linear(name, rows, outputs, width, dtype, bias=False, activation="", residual=False):
    return {"name": name, "kind": "linear", "rows": rows, "outputs": outputs, "width": width,
            "dtype": dtype, "bias": bias, "activation": activation, "residual": residual}


def _sample(name, rows, vocab, dtype, top_k=False, top_p=False, min_p=False):
    return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype,
            "top_k": top_k, "top_p": top_p, "min_p": min_p}


def _spread(rng, low, high):
    """A whole number, spread evenly over the range's logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "linear", "linear", "linear", "sample", "sample"])
    dtype = rng.choice(sorted(DTYPES))
    if kind in ("norm", "quantize"):
        width = _spread(rng, 64, 9000)
        rows = _spread(rng, 1, min(8192, 2048 * HIDDEN // width))
        if kind == "norm":
            case = _norm("", rows, width, dtype, rng.random() < 0.5)
        else:
            case = _quantize("", rows, width, dtype)
    elif kind == "sample":
        case = _sample("", _spread(rng, 1, 160), _spread(rng, 1000, 131077), dtype,
                       rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)
    else:
        width = BLOCK * _spread(rng, 1, 64)
        activation = rng.choice(["", "", "silu", "gelu", "swiglu"])
        rows = _spread(rng, 1, 2048)
        most = 2048 * 2 * HIDDEN * WIDTH // (rows * width)
        outputs = _spread(rng, 64, max(64, min(16000, most)))
        if activation == "swiglu":
            outputs += outputs % 2
        case = _linear("", rows, outputs, width, dtype, rng.random() < 0.3, activation,
                       activation != "swiglu" and rng.random() < 0.4)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"norm": _prepare_norm, "quantize": _prepare_quantize, "linear": _prepare_linear,
            "sample": _prepare_sample}[case["kind"]](case, g)


def _stream(rows, width, g):
    """Rows as a residual stream has them: of different size, a few dims of all
    rows larger."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    x *= torch.rand(rows, 1, generator=g, device="cuda") * 3 + 0.3
    return x * (1 + 9 * (torch.rand(width, generator=g, device="cuda") < 0.005))


def _prepare_norm(case, g):
    rows, width, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
    residual = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
    return {"case": case, "x": _stream(rows, width, g).to(dtype),
            "weight": 1 + 0.2 * torch.randn(width, generator=g, device="cuda"),
            "residual": residual if case["residual"] else None}


def _prepare_quantize(case, g):
    return {"case": case, "x": _stream(case["rows"], case["width"], g).to(DTYPES[case["dtype"]])}


def _prepare_linear(case, g):
    M, N, K = case["rows"], case["outputs"], case["width"]
    dev, dtype = "cuda", DTYPES[case["dtype"]]
    blocks = K // BLOCK
    # a layer as it is stored: codebooks of N(0, 0.02) quantiles that differ
    # from block to block, 3-bit indices least significant bit first
    levels = torch.tensor([-2.6, -1.07, -0.57, -0.18, 0.18, 0.57, 1.07, 2.6], device=dev)
    books = 0.02 * (levels * (1 + 0.15 * torch.randn(N, blocks, 1, generator=g, device=dev)) +
                    0.04 * torch.randn(N, blocks, ENTRIES, generator=g, device=dev))
    books = books.sort(-1).values
    index = torch.randint(0, ENTRIES, (N, K), generator=g, device=dev, dtype=torch.uint8)
    eight = index.view(N, K // 8, 8).int() << (3 * torch.arange(8, device=dev, dtype=torch.int32))
    eight = eight.sum(-1, dtype=torch.int32)
    packed = torch.stack([eight & 255, eight >> 8 & 255, eight >> 16], -1).to(torch.uint8).flatten()
    # its codebooks in 8 bits, one scale for each output, and its tiles
    scale = books.abs().amax((1, 2)) / 127
    codes = (books / scale[:, None, None]).round().clamp(-127, 127).to(torch.int8)
    # activations as rows in 8 bits
    x = _stream(M, K, g)
    x_scale = x.abs().amax(1) / 127
    x = (x / x_scale[:, None]).round().clamp(-127, 127).to(torch.int8)
    out = N // 2 if case["activation"] == "swiglu" else N
    residual = torch.randn(M, out, generator=g, device=dev).to(dtype)
    bias = 0.1 * torch.randn(N, generator=g, device=dev)
    return {"case": case, "x": x, "x_scale": x_scale, "packed": packed, "codes": codes,
            "scale": scale, "tiles": _tiles(index, codes),
            "bias": bias if case["bias"] else None,
            "residual": residual if case["residual"] else None}


def _tiles(index, codes):
    """The layout that a program makes of a layer once, when it loads it: tiles
    of 16 outputs x 128 inputs, a row's tiles one after the other; in each the
    64 units (of 32 indices in 12 bytes) of its 4 x 16 (quarter, output)s, then
    the outputs' 8 codes.  Four indices are the bytes of a selector; byte b of
    a unit's three words holds those of selectors 0 and 1, 2 and 3, 4 and 5 in
    its low six bits; the upper two hold the low bits of selectors 6 and of 7,
    in the third word the high bit of each."""
    N, K = index.shape
    blocks, tiles = K // BLOCK, (N + 15) // 16
    index = torch.nn.functional.pad(index, (0, 0, 0, tiles * 16 - N))
    codes = torch.nn.functional.pad(codes.view(N, -1), (0, 0, 0, tiles * 16 - N))
    s = index.view(tiles, 16, blocks, 4, 8, 4).permute(0, 2, 3, 1, 4, 5)   # (.., selector, byte)
    high = torch.stack([s[..., 6, :] & 3, s[..., 7, :] & 3,
                        s[..., 6, :] >> 2 | s[..., 7, :] >> 2 << 1], -2)
    units = s[..., 0:6:2, :] | s[..., 1:6:2, :] << 3 | high << 6
    codes = codes.view(tiles, 16, blocks, ENTRIES).transpose(1, 2).reshape(tiles, blocks, 128)
    return torch.cat([units.reshape(tiles, blocks, 768), codes.view(torch.uint8)], -1).contiguous()


def _prepare_sample(case, g):
    B, V, dev = case["rows"], case["vocab"], "cuda"
    # soft-capped logits; a third of the rows behind a mask that leaves half
    logits = 30 * torch.tanh(torch.randn(B, V, generator=g, device=dev) * 4 / 30)
    masked = (torch.arange(B, device=dev) % 3 == 1)[:, None] & \
        (torch.rand(B, V, generator=g, device=dev) < 0.5)

    def some(low, high):
        return torch.rand(B, generator=g, device=dev) * (high - low) + low
    top_k = (2 ** some(0, 10)).int()
    state = {"case": case, "logits": logits.masked_fill(masked, -math.inf).to(DTYPES[case["dtype"]]),
             "u": some(0, 1), "temperature": some(0.3, 1.5), "top_k": top_k, "top_p": some(0.5, 1),
             "min_p": some(0, 0.1)}
    for name in ("top_k", "top_p", "min_p"):
        state[name] = state[name] if case[name] else None
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return {"norm": _run_norm, "quantize": _run_quantize, "linear": _run_linear,
            "sample": _run_sample}[state["case"]["kind"]](state)


def _run_norm(s):
    if own:
        from nativebit_amd import ops
        if s["residual"] is None:
            return {"rows": ops.rmsnorm8(s["x"], s["weight"], 1e-6).values()}
        rows, x = ops.rmsnorm8(s["x"], s["weight"], 1e-6, residual=s["residual"])
        return {"rows": rows.values(), "x": x}
    x = s["x"]
    if s["residual"] is not None:
        x = (x.float() + s["residual"].float()).to(x.dtype)
    h = x.double()
    h = h * s["weight"].double() / (h.square().mean(1, keepdim=True) + 1e-6).sqrt()
    out = {"rows": _in_8_bits(h)}
    return out if s["residual"] is None else {**out, "x": x}


def _run_quantize(s):
    if own:
        from nativebit_amd import ops
        return ops.quantize8(s["x"]).values()
    return _in_8_bits(s["x"].double())


def _in_8_bits(x):
    """The values that codes and scales stand for, of rows in 64 bits (some
    values lie next to a border between two codes)."""
    scale = x.abs().amax(1, keepdim=True) / 127
    return torch.where(scale > 0, x / scale, 0.0).round().float() * scale.float()


def _run_linear(s):
    case = s["case"]
    M, N, K = case["rows"], case["outputs"], case["width"]
    dtype = DTYPES[case["dtype"]]
    if own:
        from nativebit_amd import ops
        return ops.linear8(ops.Rows8(s["x"], s["x_scale"]), ops.Weights8(s["tiles"], s["scale"], N, K),
                           bias=s["bias"], activation=case["activation"] or None,
                           residual=s["residual"], out_dtype=dtype)
    bits = s["packed"].view(N, K // 8, 3).int()
    eight = bits[..., 0] | bits[..., 1] << 8 | bits[..., 2] << 16
    index = (eight[..., None] >> (3 * torch.arange(8, device=bits.device)) & 7).long()
    w = s["codes"].float().view(N, K // BLOCK, ENTRIES).gather(2, index.view(N, K // BLOCK, BLOCK))
    y = s["x"].float() @ w.view(N, K).T
    y = y * (s["x_scale"][:, None] * s["scale"])
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["activation"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif case["activation"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif case["activation"] == "swiglu":
        gate, up = y[:, 0::2], y[:, 1::2]
        y = gate / (1 + torch.exp(-gate)) * up
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(dtype)


def _run_sample(s):
    if own:
        from nativebit_amd import ops
        tokens, logprobs = ops.sample(s["logits"], s["u"], temperature=s["temperature"],
                                      top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                                      logprobs=True)
        return {"tokens": tokens, "logprobs": logprobs}
    # in 64 bits: a token is chosen at a border of long sums
    x, order = s["logits"].double().sort(dim=1, descending=True, stable=True)
    B, V = x.shape
    w = torch.exp((x - x[:, :1]) / s["temperature"].double()[:, None])
    if s["top_k"] is not None:
        most = torch.where(s["top_k"] > 0, s["top_k"], V).long()
        w = w * (torch.arange(V, device=x.device) < most[:, None])
    kept = w > 0
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        upto = w.cumsum(1)
        kept &= (upto - w < p * w.sum(1, keepdim=True)) | (p >= 1)
    if s["min_p"] is not None:
        kept &= w >= s["min_p"].double()[:, None]
    w = torch.zeros_like(w).scatter_(1, order, w * kept)
    upto = w.cumsum(1)
    total = upto[:, -1:]
    tokens = (upto <= s["u"].double()[:, None] * total).sum(1).clamp(max=V - 1)
    logprobs = torch.log(w.gather(1, tokens[:, None]) / total)[:, 0]
    return {"tokens": tokens.int(), "logprobs": logprobs.float()}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    size = 2 if case["dtype"] == "bfloat16" else 4
    if kind in ("norm", "quantize"):
        n = case["rows"] * case["width"]
        # the rows in, codes and scales out, read again as the values they
        # stand for; with a residual it in and the sum out
        more = 2 * size if kind == "norm" and case["residual"] else 0
        return {"bytes": n * (size + 1.0 + 1 + 4 + more) + 4.0 * case["rows"], "flops": 6.0 * n}
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": float(n * size), "flops": 10.0 * n}
    M, N, K = case["rows"], case["outputs"], case["width"]
    out = N // 2 if case["activation"] == "swiglu" else N
    # codes of the rows and of the layer, 3 bits a weight, outputs and residuals
    return {"bytes": M * K + N * K * (3 / 8 + 8 / BLOCK) + 4.0 * (M + N) +
            M * out * size * (2.0 if case["residual"] else 1.0), "flops": 2.0 * M * N * K}


# ---------------------------------------------------------------------------
# the same from the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "quantize": _exact_quantize, "linear": _exact_linear,
            "sample": _exact_sample}[case["kind"]](s, case)


def _exact_norm(s, case):
    x = s["x"].double()
    if s["residual"] is not None:
        # (the norm is that of the sum as it is kept)
        kept = torch.add(x, s["residual"].double()).to(s["x"].dtype).double()
    else:
        kept = x
    rms = torch.linalg.vector_norm(kept, dim=1).square().div(case["width"]).add(1e-6).sqrt()
    rows = _exact_codes(kept * s["weight"].double() / rms[:, None])
    return {"rows": rows} if s["residual"] is None else {"rows": rows, "x": x + s["residual"].double()}


def _exact_quantize(s, case):
    return _exact_codes(s["x"].double())


def _exact_codes(v):
    step = torch.linalg.vector_norm(v, ord=math.inf, dim=1, keepdim=True) / 127
    return torch.round(v / step) * step


def _exact_linear(s, case):
    M, N, K = case["rows"], case["outputs"], case["width"]
    # bit j of weight i is bit 3 i + j of the stream
    at = 3 * torch.arange(K, device="cuda")[:, None] + torch.arange(3, device="cuda")
    out = torch.empty(M, N, dtype=torch.float64, device="cuda")
    x = s["x"].double() * s["x_scale"].double()[:, None]
    rows = s["packed"].view(N, K * 3 // 8)
    for n in range(0, N, 512):
        bit = rows[n:n + 512, at // 8] >> (at % 8).to(torch.uint8) & 1
        entry = bit[..., 0].long() + 2 * bit[..., 1] + 4 * bit[..., 2]
        count = entry.shape[0]
        block = torch.arange(K, device="cuda") // BLOCK
        books = s["codes"][n:n + 512].double() * s["scale"][n:n + 512].double()[:, None, None]
        w = books[torch.arange(count, device="cuda")[:, None], block, entry]
        out[:, n:n + 512] = x @ w.T.contiguous()
    if s["bias"] is not None:
        out += s["bias"].double()
    if case["activation"] == "silu":
        out = torch.sigmoid(out) * out
    elif case["activation"] == "gelu":
        out = out * 0.5 * torch.special.erfc(-out / math.sqrt(2))
    elif case["activation"] == "swiglu":
        pairs = out.view(M, N // 2, 2)
        out = torch.sigmoid(pairs[..., 0]) * pairs[..., 0] * pairs[..., 1]
    return out if s["residual"] is None else out + s["residual"].double()


def _exact_sample(s, case):
    """Row by row: the tokens are whole numbers, their log-probabilities are
    those of the tokens that 64 bits draw."""
    import numpy as np
    x, u, t = (s[k].double().cpu().numpy() for k in ("logits", "u", "temperature"))
    logprobs = np.empty(x.shape[0])
    for b, row in enumerate(x):
        ids = np.lexsort((np.arange(row.size), -row))
        ids = ids[np.isfinite(row[ids])]
        if s["top_k"] is not None and s["top_k"][b] > 0:
            ids = ids[:int(s["top_k"][b])]
        z = row[ids] / t[b]
        p = np.exp(z - z.max())
        share = p / math.fsum(p)
        keep = np.ones(ids.size, bool)
        if s["top_p"] is not None and s["top_p"][b] < 1:
            keep[1:] &= np.cumsum(share)[:-1] < float(s["top_p"][b])
        if s["min_p"] is not None:
            keep &= p >= float(s["min_p"][b])
        ids, share = ids[keep], share[keep]
        at = np.argsort(ids)
        upto = np.cumsum(share[at])
        i = min(int(np.searchsorted(upto, u[b] * upto[-1], side="right")), ids.size - 1)
        logprobs[b] = math.log(share[at][i] / upto[-1])
    return {"tokens": None, "logprobs": torch.from_numpy(logprobs)}
