"""Plain restatements, in 64 bits or more on the host, of rows in 8 bits, of
their products with packed layers and of drawn tokens."""
import math

import numpy as np
import torch


def codes(v):
    """(codes, a) of float64 rows: rint(v * (127 / a)), a the row's largest
    magnitude; rows that are not finite have codes 0 and a = nan."""
    a = np.abs(v).max(1)
    a = np.where(np.isfinite(v).all(1), a, np.nan)
    turn = np.where(a > 0, 127.0 / np.where(a > 0, a, 1.0), 0.0)
    with np.errstate(invalid="ignore"):
        q = np.rint(v * turn[:, None])
    return np.where(np.isfinite(a)[:, None], q, 0).astype(np.int8), a


def quantize8(x):
    """(codes, scale) of a tensor's rows."""
    q, a = codes(x.double().numpy())
    return q, (a / 127.0).astype(np.float32)


def rmsnorm8(x, weight, eps, residual=None):
    """(codes, scale in 64 bits, sum) of tensors."""
    if residual is not None:
        x = (x.float() + residual.float()).to(x.dtype)
    h = x.double().numpy()
    with np.errstate(invalid="ignore", over="ignore"):
        q, a = codes(h * weight.double().numpy())
        rms = np.sqrt((h * h).mean(1) + np.float64(np.float32(eps)))
        scale = np.where(a == 0, 0.0, a / np.where(a == 0, 1.0, 127.0 * rms))
    return q, scale, x


def layer8(codebook):
    """(codes, scale) of a layer's (N, blocks, 8) float32 codebooks."""
    n = codebook.shape[0]
    q, a = codes(codebook.reshape(n, -1).astype(np.float64))
    return q.reshape(codebook.shape), (a / 127.0).astype(np.float32)


def tiles(index, q):
    """The tiles of (N, K) indices and (N, blocks, 8) codes, byte by byte."""
    N, K = index.shape
    nb, nt = K // 128, -(-N // 16)
    out = np.zeros((nt, nb, 896), np.uint8)
    for n in range(N):
        t, r = divmod(n, 16)
        for j in range(nb):
            out[t, j, 768 + 8 * r:776 + 8 * r] = q[n, j].view(np.uint8)
            for g in range(4):
                at = 12 * (16 * g + r)
                i = index[n, 128 * j + 32 * g:128 * j + 32 * g + 32].reshape(8, 4).astype(np.int64)
                words = np.stack([i[0] | i[1] << 3 | (i[6] & 3) << 6, i[2] | i[3] << 3 | (i[7] & 3) << 6,
                                  i[4] | i[5] << 3 | (i[6] >> 2) << 6 | (i[7] >> 2) << 7])
                out[t, j, at:at + 12] = words.astype(np.uint8).reshape(-1)
    return out.reshape(-1)


def linear8(x, x_scale, index, q, scale, bias, activation, residual, dtype, dev="cpu"):
    """(outputs in 64 bits, how far fp32 steps may be off) on the host; the
    products on `dev`."""
    N, K = index.shape
    w = np.take_along_axis(q, index.reshape(N, K // 128, 128).astype(np.int64), 2).reshape(N, K)
    # whole numbers under 2^31: exact in 64 bits, in any order
    sums = torch.matmul(torch.from_numpy(x).to(dev).double(),
                        torch.from_numpy(w).to(dev).double().T.contiguous()).cpu().numpy()
    v = sums * x_scale.astype(np.float64)[:, None] * scale.astype(np.float64)
    h = 2.0 ** -24                                           # half a step of fp32
    # the sum as fp32, the scales' product, their product
    off = 3.01 * h * np.abs(v)
    if bias is not None:
        v = v + bias.astype(np.float64)
        off = off + h * np.abs(v) + h * off

    def silu(z, oz):
        s = z / (1 + np.exp(-z))
        # |silu'| <= 1.1; exp: its argument's rounding times |z|, a step of its own
        return s, 1.1 * oz + np.abs(s) * ((np.abs(z) + 2) * 2 * h + 3 * h)
    if activation == "silu":
        v, off = silu(v, off)
    elif activation == "gelu":
        s = 0.5 * v * torch.special.erfc(torch.from_numpy(-v / math.sqrt(2))).numpy()
        # |gelu'| <= 1.13; erfc within 16 steps, its argument's two roundings times
        # its condition (under 2 + v^2)
        v, off = s, 1.13 * off + np.abs(s) * (16 + 2 * (2 + v * v) + 2) * 2 * h
    elif activation == "swiglu":
        s, os = silu(v[:, 0::2], off[:, 0::2])
        u, ou = v[:, 1::2], off[:, 1::2]
        v, off = s * u, np.abs(u) * os + np.abs(s) * ou + os * ou + h * np.abs(s * u)
    if residual is not None:
        v = v + residual.astype(np.float64)
        off = off + h * (np.abs(v) + off)
    if dtype == torch.bfloat16:
        off = off + 2.0 ** -8 * (np.abs(v) + off)
    return v, off + 1e-37


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob) of one row of float32 or bfloat16 logits, in extended
    precision."""
    x = row.double().numpy()
    V = x.size
    ids = [v for v in sorted(range(V), key=lambda v: (-x[v] if x[v] == x[v] else math.inf, v))
           if x[v] > -math.inf]
    if not ids:
        return -1, -math.inf
    most = x[ids[0]]
    if not temperature > 0:
        return ids[0], 0.0
    ld = np.longdouble
    with np.errstate(all="ignore"):
        w = np.array([ld(1) if x[v] == most else np.exp(max((ld(x[v]) - ld(most)) / ld(temperature), ld(-5000)))
                      if math.isfinite(most) else ld(0) for v in ids])
    if 0 < top_k < len(ids):
        ids, w = ids[:top_k], w[:top_k]
    if top_p < 1:
        before = np.cumsum(w) - w
        keep = before < ld(max(top_p, 0.0)) * w.sum()
        keep[0] = True
        ids, w = [v for v, k in zip(ids, keep) if k], w[keep]
    if min_p > 0:
        keep = w >= ld(min(min_p, 1.0))
        ids, w = [v for v, k in zip(ids, keep) if k], w[keep]
    order = np.argsort(ids)
    ids, w = np.array(ids)[order], w[order]
    upto = np.cumsum(w)
    at = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    i = int(np.searchsorted(upto, ld(at) * upto[-1], side="right"))
    i = min(i, len(ids) - 1)
    return int(ids[i]), float(np.log(w[i] / upto[-1]))
