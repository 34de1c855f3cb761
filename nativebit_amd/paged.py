"""Serving several requests of different lengths with one 8-bit key / value
cache: the cache, and greedy generation over it.

``PagedCache`` holds, for every layer of a ``PackedGPT``, blocks of 64 tokens
(int8 codes, one fp32 scale for each block and head) that the requests share:
a request takes blocks as it grows and gives them back when it ends.  A step
is ``cache.step(new)`` -- how many tokens each request brings -- and a forward
pass over those tokens' rows, the requests' one after the other:

    cache = PagedCache(model, n_blocks=400, max_requests=16)
    cache.step([len(p) for p in prompts])
    logits, _ = model(torch.tensor([sum(prompts, [])], device="cuda"), kv_caches=cache)

The reference has one fp32 cache of fixed shape for each sequence
(inference/generate_torch.py:269-277) and decodes one sequence at a time
(298-313).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import ops


class PagedLayer(NamedTuple):
    """One layer of a PagedCache, as an attention module takes it for its
    ``kv_cache``."""
    cache: "PagedCache"
    index: int

    def attend(self, qkv, cos, sin, n_head):
        """Attention of the step's rows, (rows, q | k | v) float32, over their
        requests' cached tokens, their own appended first; float32, 0 in the
        rows that the step has no slot for."""
        c, i = self.cache, self.index
        if c.plan is None or qkv.shape[0] != c.plan.slots.shape[0]:
            planned = "no step" if c.plan is None else f"a step of {c.plan.slots.shape[0]} rows"
            raise ValueError(f"{qkv.shape[0]} rows for a cache with {planned} planned")
        store = (c.k[i], c.v[i], c.k_scale[i], c.v_scale[i])
        rows = torch.empty if c.whole else torch.zeros
        q = rows(qkv.shape[0], n_head * c.head_dim, device=qkv.device)
        out = rows(qkv.shape[0], n_head * c.head_dim, device=qkv.device)
        ops.kv8_append(qkv, c.plan, cos, sin, *store, n_head, q=q)
        return ops.kv8_attention(q, c.plan, c.table, *store, softcap=c.softcap, window=c.window,
                                 slopes=c.slopes, prefix=c.prefix, out=out)


class PagedCache:
    """The 8-bit block cache of a PackedGPT for up to ``max_requests`` requests
    of up to ``max_len`` tokens (the model's context by default), ``n_blocks``
    blocks of 64 tokens in all.  ``softcap``, ``window`` and ``slopes`` (one
    for each head) change every layer's attention as in ops.kv8_attention.

    ``table``, ``lens``, ``free`` and ``state`` are the block tables, lengths,
    free list and (free blocks, tokens of the last step without a slot) on the
    GPU."""

    def __init__(self, model, n_blocks: int, max_requests: int, max_len: int | None = None, *,
                 softcap: float = 0.0, window: int = 0, slopes=None, device="cuda"):
        H, D = model.n_head, model.n_embd // model.n_head
        max_len = model.context_len if max_len is None else int(max_len)
        if n_blocks < 1 or max_requests < 1 or not 1 <= max_len <= model.context_len:
            raise ValueError(f"n_blocks={n_blocks}, max_requests={max_requests}, max_len={max_len} "
                             f"(context {model.context_len})")
        if D % 16 or not 16 <= D <= 256:
            raise ValueError(f"head_dim {D}: the 8-bit cache takes multiples of 16 up to 256")
        L, B = model.n_layers, ops.KV_BLOCK
        self.n_layers, self.head_dim, self.max_len = L, D, max_len
        self.softcap, self.window = float(softcap), int(window)
        self.slopes = None if slopes is None else \
            torch.as_tensor(slopes, dtype=torch.float32).to(device).contiguous()

        def zeros(*shape, dtype=torch.int32):
            return torch.zeros(*shape, dtype=dtype, device=device)
        self.k = zeros(L, n_blocks, H, B, D, dtype=torch.int8)
        self.v = zeros(L, n_blocks, H, D, B, dtype=torch.int8)
        self.k_scale = zeros(L, n_blocks, H, dtype=torch.float32)
        self.v_scale = zeros(L, n_blocks, H, dtype=torch.float32)
        self.table = zeros(max_requests, -(-max_len // B)) - 1
        self.lens = zeros(max_requests)
        self.free = torch.arange(n_blocks - 1, -1, -1, dtype=torch.int32, device=device)
        self.state = torch.tensor([n_blocks, 0], dtype=torch.int32, device=device)
        self.plan = self.prefix = None
        self.whole = True           # every row of the step has a slot
        self._known = [0] * max_requests    # the lengths, where the host knows them
        self._left = n_blocks
        self._captured = False      # whether replays may change them unseen

    def __len__(self):
        return self.n_layers

    def __getitem__(self, i) -> PagedLayer:
        if not 0 <= i < self.n_layers:
            raise IndexError(i)
        return PagedLayer(self, i)

    def step(self, new, n_tokens: int | None = None, prefix=None):
        """Plans a step in which request r brings ``new[r]`` tokens (fewer
        entries than requests: the others bring none).  A list is checked here:
        it raises where a request grows past max_len or the blocks do not
        suffice, and the step's rows are its sum.  An int32 GPU tensor
        (max_requests,) is not read on the host (a step of ``n_tokens`` rows,
        which may be captured in a graph); tokens that no room is left for have
        no slot then, and ``state[1]`` counts them.  (After a captured step
        lists read the lengths back from the GPU: replays change them.)
        ``prefix``: for each request a number of leading tokens that all its
        queries see.  With slopes it takes a list, and no new token may have
        others behind it in its prefix: their bias would grow with the distance."""
        R = self.table.shape[0]
        dev = self.table.device
        ahead = None
        if prefix is not None:
            prefix = torch.as_tensor(prefix, dtype=torch.int32).to(dev)
            if prefix.shape != (R,):
                raise ValueError(f"prefix must have {R} numbers, got {tuple(prefix.shape)}")
            if self.slopes is not None:
                if isinstance(new, torch.Tensor):
                    raise ValueError("slopes and a prefix take a step from a list (which tokens lie "
                                     "inside a prefix is checked on the host)")
                ahead = prefix.tolist()
        whole = not isinstance(new, torch.Tensor)
        known = left = None
        if whole:
            new = [int(n) for n in new]
            if len(new) > R or min(new, default=0) < 0:
                raise ValueError(f"{len(new)} counts for {R} requests, none below 0")
            if n_tokens is not None and n_tokens != sum(new):
                raise ValueError(f"n_tokens={n_tokens}, {sum(new)} tokens")
            new += [0] * (R - len(new))
            if self._known is None or self._captured:   # (lengths that only the GPU knows)
                self._known, self._left = self.lens.tolist(), int(self.state[0])
            known = [a + b for a, b in zip(self._known, new)]
            need = sum(-(-e // ops.KV_BLOCK) - -(-a // ops.KV_BLOCK)
                       for a, e in zip(self._known, known))
            if max(known) > self.max_len:
                raise ValueError(f"{max(known)} tokens of a request exceed max_len {self.max_len}")
            if need > self._left:
                raise ValueError(f"{need} blocks needed, {self._left} free")
            if ahead is not None:
                for r, (a, e, p) in enumerate(zip(self._known, known, ahead)):
                    if e > a and min(p, e) > a + 1:   # its first token sees others behind it
                        raise ValueError(f"slopes with tokens of request {r} inside its prefix: "
                                         "their bias would grow past the query")
            left = self._left - need
            n_tokens = sum(new)
            new = torch.tensor(new, dtype=torch.int32, device=dev)
        elif n_tokens is None:
            raise ValueError("a step from a tensor needs n_tokens")
        elif self.table.is_cuda and torch.cuda.is_current_stream_capturing():
            self._captured = True
        plan = ops.kv_plan(self.table, self.lens, new, self.free, self.state, n_tokens,
                           max_len=self.max_len)
        self.lens.copy_(plan.lens)
        self.state.copy_(plan.state)
        self.plan, self.prefix, self.whole = plan, prefix, whole
        self._known, self._left = known, left
        return plan

    def release(self, requests) -> None:
        """Ends requests (their numbers): their blocks are free again."""
        R = self.table.shape[0]
        requests = sorted({int(r) for r in requests})
        if requests and not 0 <= requests[0] <= requests[-1] < R:
            raise ValueError(f"requests {requests} of {R}")
        finished = torch.zeros(R, dtype=torch.int32)
        finished[requests] = 1
        ops.kv_release(self.table, self.lens, finished.to(self.table.device), self.free, self.state)
        self.plan = None    # (its lengths and slots are the ended requests' too)
        if self._captured:
            self._known = None
        if self._known is not None:
            for r in requests:
                self._left += -(-self._known[r] // ops.KV_BLOCK)
                self._known[r] = 0

    def read(self, layer: int, request: int):
        """The (keys, values) that a request has cached in a layer, float32
        (heads, tokens, head_dim), the shape of the reference's caches."""
        n = int(self.lens[request])
        j = torch.arange(n, device=self.table.device)
        slots = self.table[request, j // ops.KV_BLOCK] * ops.KV_BLOCK + j % ops.KV_BLOCK
        keys, values = ops.kv8_read(slots.int(), self.k[layer], self.v[layer],
                                    self.k_scale[layer], self.v_scale[layer])
        return keys.transpose(0, 1), values.transpose(0, 1)


def _per_request(x, n, device):
    """A number for all requests, or one for each, as a float32 tensor."""
    if x is None:
        return None
    t = torch.as_tensor(x, dtype=torch.float32)
    return (t.expand(n) if t.dim() == 0 else t).contiguous().to(device)


@torch.no_grad()
def generate(model, prompts, n_generate: int, *, repetition=None, frequency=None, presence=None,
             bias=None, mask=None, cache: PagedCache | None = None):
    """Greedy continuations of several prompts at once, ``n_generate`` tokens
    each: the prompts as one ragged pass, then one token of every request a
    step, chosen by ops.logits_rules.  ``repetition``, ``frequency`` and
    ``presence``: a number or one for each request; ``bias``: a dict token ->
    bias for each request; ``mask``: int32 (requests, vocabulary / 32) bit
    masks of the allowed tokens.  A request whose mask and biases leave no
    token gets -1 (fed as token 0).  ``cache``: an empty cache to use, with room
    for all requests to their ends; they stay in it."""
    prompts = [[int(t) for t in p] for p in prompts]
    n = len(prompts)
    if not n or not all(prompts) or n_generate < 0:
        raise ValueError("prompts must hold a token each")
    V = model.embedding.weight.shape[0]
    if min(map(min, prompts)) < 0 or max(map(max, prompts)) >= V:
        raise ValueError(f"prompt token outside 0..{V - 1}")
    dev = model.embedding.weight.device
    lengths = [len(p) for p in prompts]
    room = model.context_len if cache is None else cache.max_len
    if max(lengths) + n_generate - 1 > room:     # (the last token is not fed)
        raise ValueError(f"{max(lengths)} prompt tokens and {n_generate} more exceed {room}")
    if bias is not None and len(bias) != n:
        raise ValueError(f"{len(bias)} bias dicts for {n} prompts")
    if cache is not None and bool(cache.lens.any()):
        raise ValueError("the cache holds requests already")
    if cache is not None and n_generate:
        blocks = sum(-(-(length + n_generate - 1) // ops.KV_BLOCK) for length in lengths)
        if n > cache.table.shape[0] or blocks > int(cache.state[0]):
            raise ValueError(f"{n} requests of {blocks} blocks, the cache is for "
                             f"{cache.table.shape[0]} and has {int(cache.state[0])} free")
    if cache is None:
        blocks = sum(-(-(length + n_generate) // ops.KV_BLOCK) for length in lengths)
        cache = PagedCache(model, blocks, n, device=dev)
    if n_generate == 0:
        return [[] for _ in prompts]
    width = max(lengths) + n_generate
    history = torch.tensor([p + [-1] * (width - len(p)) for p in prompts], dtype=torch.int32, device=dev)
    prompt_lens = torch.tensor(lengths, dtype=torch.int32, device=dev)
    lens = prompt_lens.clone()
    rules = {"history": history, "lens": lens, "prompt_lens": prompt_lens, "mask": mask,
             "repetition": _per_request(repetition, n, dev),
             "frequency": _per_request(frequency, n, dev),
             "presence": _per_request(presence, n, dev)}
    if bias is not None:
        most = max((len(b) for b in bias), default=0)
        rules["bias_ids"] = torch.tensor([list(b) + [-1] * (most - len(b)) for b in bias],
                                         dtype=torch.int32, device=dev).view(n, most)
        rules["bias"] = torch.tensor([list(b.values()) + [0.0] * (most - len(b)) for b in bias],
                                     dtype=torch.float32, device=dev).view(n, most)
    idx = torch.tensor([sum(prompts, [])], device=dev)
    rows = torch.tensor(lengths, device=dev).cumsum(0) - 1     # of the requests' last tokens
    cache.step(lengths)
    out = []
    for i in range(n_generate):
        hidden, _ = model.hidden(idx, cache)
        logits = model.head(hidden[0, rows])
        _, tokens = ops.logits_rules(logits.contiguous(), out=logits, choose=True, **rules)
        out.append(tokens)
        if i + 1 == n_generate:
            break
        history.scatter_(1, lens.long()[:, None], tokens[:, None])
        lens += 1
        idx = tokens.clamp(min=0).long()[None]
        if i == 0:
            rows = torch.arange(n, device=dev)
        cache.step([1] * n)
    return torch.stack(out, 1).tolist()
