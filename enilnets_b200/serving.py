"""Batched serving over a paged key-value cache.

The reference decodes one cache per batch (nn/kvcache.py:23-120): every row of
it has the same length, so its TextGenerator groups prompts by token count
(generative/text_generation.py:315-381). Here any sequences share one pool of
pages: `PagedKVCache` hands pages to sequences as they grow and takes them back
when they end, `paged_forward_step` runs one step of a ragged batch through a
model's layers, and `sample` draws the next tokens on the device.

One step of one attention layer is the projection (K6), the queries' and keys'
norm and rotation together with the append into the pages (one kernel), and the
attention over the pages (one kernel for single tokens, K1 for prompts). Lengths,
tables and drawn tokens stay on the device between the kernels of a step; the
host keeps its own copy of the lengths, which it knows without asking.
"""
from __future__ import annotations

from typing import Any, Dict, List, Optional, Sequence

import numpy as np

from . import attention, kernels
from .backend import WEIGHTS, device, to_device
from .network import dense, embed, layernorm, positional_table


class PagedKVCache:
    """Pages of keys and values shared by sequences of any lengths.

    num_pages pages of page_size positions each, per attention layer (the
    layers' pools are made when a layer is first stepped, (num_pages, kv_heads,
    page_size, head_dim) in the compute dtype); max_seq_len bounds one sequence.
    window, sinks: single-token steps see only the last `window` positions before
    the query and the first `sinks` (None: all), and pages that no later step can
    see go back to the pool, so that a stream of any length up to max_seq_len holds
    a bounded number of them.
    """

    def __init__(self, num_pages: int, page_size: int = 16, max_seq_len: int = 4096,
                 window: Optional[int] = None, sinks: int = 0) -> None:
        if num_pages < 1 or page_size < 1 or max_seq_len < 1:
            raise ValueError(f"num_pages={num_pages}, page_size={page_size} and "
                             f"max_seq_len={max_seq_len} must be >= 1")
        if sinks < 0 or (window is not None and window < 0) or (sinks and window is None):
            raise ValueError(f"window={window} and sinks={sinks}: sinks need a window, neither "
                             "may be negative")
        self.num_pages, self.page_size = int(num_pages), int(page_size)
        self.max_seq_len = int(max_seq_len)
        self.window, self.sinks = window, int(sinks)
        self.pools: Dict[int, tuple] = {}
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._pages: Dict[int, List[int]] = {}  # sequence -> page numbers, -1: given back
        self.length: Dict[int, int] = {}
        self._next = 0

    @staticmethod
    def pages_held(prompt: int, total: int, page_size: int, window: Optional[int] = None,
                   sinks: int = 0) -> int:
        """The most pages a sequence holds at once that starts with `prompt` positions
        in one step and grows by single tokens to `total`."""
        all_of_it = -(-total // page_size)
        if window is None:
            return all_of_it
        # A step holds the first tokens' pages and those of the last window + 1 positions.
        step = -(-sinks // page_size) + -(-window // page_size) + 1
        return min(all_of_it, max(-(-prompt // page_size), step))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def add(self) -> int:
        """A new, empty sequence; returns its handle."""
        seq = self._next
        self._next += 1
        self._pages[seq] = []
        self.length[seq] = 0
        return seq

    def release(self, seq: int) -> None:
        """End a sequence; its pages go back to the pool."""
        if seq not in self._pages:
            raise ValueError(f"sequence {seq} is not in this cache")
        self._free.extend(p for p in self._pages.pop(seq) if p >= 0)
        del self.length[seq]

    def reserve(self, seqs: Sequence[int], n_new: Sequence[int]) -> None:
        """Pages for n_new[i] more positions of each sequence; raises ValueError
        (and takes none) when a sequence would pass max_seq_len or the pool has too
        few left."""
        need = []
        for s, n in zip(seqs, n_new):
            if s not in self._pages:
                raise ValueError(f"sequence {s} is not in this cache")
            total = self.length[s] + int(n)
            if total > self.max_seq_len:
                raise ValueError(f"sequence {s} would hold {total} positions, more than "
                                 f"max_seq_len={self.max_seq_len}")
            need.append(max(0, -(-total // self.page_size) - len(self._pages[s])))
        if sum(need) > len(self._free):
            raise ValueError(f"the cache needs {sum(need)} more pages and has {len(self._free)} "
                             f"of {self.num_pages} left")
        for s, n in zip(seqs, need):
            self._pages[s].extend(self._free.pop() for _ in range(n))

    def advance(self, seqs: Sequence[int], n_new: Sequence[int]) -> None:
        """Count n_new[i] positions as cached, and give back the pages that a
        windowed cache's later steps cannot see."""
        for s, n in zip(seqs, n_new):
            self.length[s] += int(n)
            if self.window is None:
                continue
            # The next query sits at length; it sees from length - window on.
            first_seen = max(0, self.length[s] - self.window)
            pages = self._pages[s]
            keep_first = -(-self.sinks // self.page_size)
            for i in range(keep_first, min(len(pages), first_seen // self.page_size)):
                if pages[i] >= 0:
                    self._free.append(pages[i])
                    pages[i] = -1

    def table(self, seqs: Sequence[int]):
        """int32 (len(seqs), max pages of these) block table on the device. Pages
        given back are entered as page 0, which no step reads for them."""
        import torch
        cols = max(1, max((len(self._pages[s]) for s in seqs), default=1))
        host = np.zeros((len(seqs), cols), dtype=np.int32)
        for i, s in enumerate(seqs):
            host[i, :len(self._pages[s])] = np.maximum(self._pages[s], 0)
        return to_device(host, torch.int32)

    def pool(self, idx: int, Hkv: int, D: int, dtype):
        """(k_pages, v_pages) of layer idx."""
        import torch
        have = self.pools.get(idx)
        if have is None:
            shape = (self.num_pages, Hkv, self.page_size, D)
            have = self.pools[idx] = (torch.zeros(shape, dtype=dtype, device=device()),
                                      torch.zeros(shape, dtype=dtype, device=device()))
        elif have[0].dtype != dtype:
            raise ValueError(f"the cache of layer {idx} holds {have[0].dtype} pages but the "
                             f"precision is now {dtype}; start a new PagedKVCache")
        return have


class _Step:
    """What the layers of one step share."""

    def __init__(self, cache: PagedKVCache, seqs: Sequence[int], n_new: Sequence[int]) -> None:
        import torch
        self.cache, self.seqs = cache, list(seqs)
        self.start = [cache.length[s] for s in self.seqs]
        self.n_new = [int(n) for n in n_new]
        self.width = max(self.n_new)
        i32 = lambda v: to_device(np.asarray(v, dtype=np.int32), torch.int32)  # noqa: E731
        self.table = cache.table(self.seqs)
        self.start_t = i32(self.start)
        self.n_new_t = None if min(self.n_new) == self.width else i32(self.n_new)
        self.lens_t = i32([a + n for a, n in zip(self.start, self.n_new)])


def _check_layer(layer: Dict[str, Any], idx: int, cache: PagedKVCache) -> None:
    if not layer.get("causal", False):
        raise ValueError(f"paged stepping requires causal attention; layer {idx} is non-causal")
    attention.check_supported(layer)
    if layer.get("attention_kernel", "softmax") != "softmax" or \
            layer.get("sparse_pattern") is not None:
        raise ValueError(f"paged stepping covers softmax layers without a sparse_pattern (layer "
                         f"{idx})")


def _attention(layer: Dict[str, Any], x, idx: int, step: _Step):
    """One attention layer's step on the paged cache: (B, S, E) -> (B, S, E) fp32."""
    import torch
    cache = step.cache
    _check_layer(layer, idx, cache)
    H, D = layer["num_heads"], layer["head_dim"]
    Hkv = layer.get("num_kv_heads") or H
    qkv = attention.project(x, layer, "qkv")
    q = attention.split_heads(qkv, H, D, 0)
    k = attention.split_heads(qkv, Hkv, D, H * D)
    v = attention.split_heads(qkv, Hkv, D, H * D + Hkv * D)
    kp, vp = cache.pool(idx, Hkv, D, qkv.dtype)
    wq, wk, eps = attention.qk_norm_args(layer)
    scheme = layer.get("positional_scheme", "absolute")
    rope = None
    if scheme == "rope":
        rope = attention.rope_tables(max(a + step.width for a in step.start), D)
    slopes = attention.alibi_tensor(H) if scheme == "alibi" else None
    q = kernels.qk_norm_rope_append(q, k, v, kp, vp, step.table, step.start_t, n_new=step.n_new_t,
                                    q_weight=wq, k_weight=wk, eps=eps, rope=rope)
    window, sinks = layer.get("window_size"), 0
    if step.width == 1:
        if cache.window is not None and (window is None or window > cache.window):
            window, sinks = cache.window, cache.sinks
        ctx = kernels.attention_decode_paged(q[:, 0], kp, vp, step.table, step.lens_t,
                                             window=window, sinks=sinks,
                                             alibi_slopes=slopes).unsqueeze(1)
    else:
        # Prompts: each row's cached positions as one contiguous stretch, K1 with
        # the row's own offset.
        if cache.window is not None and max(step.start) > cache.window:
            raise ValueError("a windowed cache takes several tokens at a time only while it "
                             "still holds every position")
        ctx = torch.zeros_like(q)
        for i, (a, n) in enumerate(zip(step.start, step.n_new)):
            if n == 0:
                continue
            pages = step.table[i, :-(-(a + n) // cache.page_size)].long()
            ki, vi = (t[pages].permute(0, 2, 1, 3).reshape(1, -1, Hkv, D)[:, :a + n]
                      for t in (kp, vp))
            ctx[i:i + 1, :n] = kernels.attention_prefill(
                q[i:i + 1, :n], ki, vi, causal=True, window=window, alibi_slopes=slopes,
                q_pos0=a, out_dtype=q.dtype)
    return attention.project(ctx.flatten(-2), layer, "o", out_dtype=torch.float32)


def paged_forward_step(model: Any, tokens: Sequence[Sequence[int]], cache: PagedKVCache,
                       seqs: Sequence[int]):
    """One step of a ragged batch: tokens[i] are the new tokens of sequence
    seqs[i], any number of them each (a prompt, or the one token drawn last).
    Returns the logits of each sequence's newest token, (len(seqs), out_dim) fp32
    on the device: the last layer's output before its softmax."""
    import torch
    n_new = [len(t) for t in tokens]
    if len(tokens) != len(seqs) or not len(seqs) or len(set(seqs)) != len(seqs) or min(n_new) < 1:
        raise ValueError("paged_forward_step needs one or more tokens for each of one or more "
                         f"different sequences (got {n_new} for {list(seqs)})")
    cache.reserve(seqs, n_new)
    step = _Step(cache, seqs, n_new)
    B, S = len(seqs), step.width
    ids = np.zeros((B, S), dtype=np.int64)
    for i, t in enumerate(tokens):
        ids[i, :len(t)] = t
    x: Any = ids
    saved: Dict[int, Any] = {}
    last = len(model.layers) - 1
    newest = to_device(np.asarray(n_new, dtype=np.int64) - 1, torch.int64)
    rows = torch.arange(B, device=device())
    for idx, layer in enumerate(model.layers):
        t = layer["type"]
        if t == "embedding":
            x = embed(x, layer)
        elif t == "positional_encoding":
            table = positional_table(layer)
            if max(a + n for a, n in zip(step.start, n_new)) > table.shape[0]:
                raise ValueError(f"positions exceed the positional table ({table.shape[0]} rows) "
                                 f"of layer {idx}")
            at = step.start_t.long()[:, None] + torch.arange(S, device=x.device)
            x = x + table[at.clamp(max=table.shape[0] - 1)]
        elif t == "layernorm":
            x = layernorm(x, layer)
        elif t in ("dense", "sparse"):
            if idx == last:
                x = x[rows, newest]  # only the newest tokens' logits are wanted
                if layer["activation"] == "softmax":
                    x = x @ WEIGHTS.get(layer["weights"], torch.float32).T + \
                        WEIGHTS.get(layer["bias"], torch.float32)
                else:
                    x = torch.log(dense(x, layer).clamp_min(1e-30))
                break
            x = dense(x, layer)
        elif t == "dropout":
            pass                                        # inference no-op
        elif t == "residual_save":
            saved[idx] = x
        elif t == "residual_add":
            x = x + saved[layer["save_index"]]
        elif t == "multihead_attention":
            x = _attention(layer, x, idx, step)
        else:
            raise ValueError(f"paged stepping doesn't support layer type '{t}' (layer {idx})")
    else:
        x = x[rows, newest]
    cache.advance(seqs, n_new)
    return x


def sample(logits, u, temperature: float = 1.0, top_p: Optional[float] = None,
           top_k: Optional[int] = None, min_p: Optional[float] = None,
           greedy: bool = False) -> List[int]:
    """Token ids drawn from logits (B, V) with the uniform numbers u (B,), one
    device call and one copy of B numbers back. Raises ValueError when a row has
    no logit to draw from (all of them NaN or -inf)."""
    import torch
    out = kernels.sample_tokens(
        logits, to_device(np.asarray(u, dtype=np.float32), torch.float32),
        temperature=0.0 if greedy else float(temperature), top_k=top_k, top_p=top_p, min_p=min_p)
    tokens = out.tolist()
    dead = [b for b, t in enumerate(tokens) if t < 0]
    if dead:
        raise ValueError(f"no token to draw in rows {dead}: every logit is NaN or -inf")
    return tokens
