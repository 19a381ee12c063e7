"""Measured cases of the operators of one serving step over a paged key-value cache (and of the
training pass of its first one):

* rope:    per-head RMS norm of queries and keys with the position rotation, forward and backward
* append:  its serving form, which also writes the new keys and values into the cache's pages
* decode:  attention of one new token over the pages
* sample:  the next token from logits, with temperature, top-k, top-p and min-p

`own` false computes the plain forms below, true calls the framework.
"""
import math

import torch

own = False

EPS = 1e-6
ROPE_BASE = 10000.0
WEIGHT_ONE = float(1 << 40)  # fixed point of the sampling weights: whole numbers, so sums are exact
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp32": 4}


# ------------------------------------------------------------------ cases
def _rope(name, batch, seq, heads, kv_heads, dim, dtype, grad, pos0=0):
    return {"name": name, "op": "rope", "batch": batch, "seq": seq, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "grad": grad, "pos0": pos0}


def _append(name, batch, seq, heads, kv_heads, dim, dtype, page, max_start, norm=True):
    return {"name": name, "op": "append", "batch": batch, "seq": seq, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page,
            "max_start": max_start, "norm": norm}


def _decode(name, batch, heads, kv_heads, dim, dtype, page, min_len, max_len, window=-1, sinks=0):
    return {"name": name, "op": "decode", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "dtype": dtype, "page": page, "min_len": min_len, "max_len": max_len,
            "window": window, "sinks": sinks}


def _sample(name, batch, vocab, dtype, kind):
    return {"name": name, "op": "sample", "batch": batch, "vocab": vocab, "dtype": dtype,
            "kind": kind}


def listed():
    return [
        # One decode step of a small batch: the smallest call, where latency counts.
        _append("append, 8 new tokens", 8, 1, 32, 8, 128, "bf16", 16, 8191),
        # Prompts of unequal lengths entering the cache in the default float32 precision.
        _append("append, ragged prompts fp32", 5, 1021, 16, 4, 64, "fp32", 24, 300),
        # Training forward at the causal prefill's size (batch 8, 4096 tokens, 16 heads of 128).
        _rope("norm+rope, training forward", 8, 4096, 16, 16, 128, "bf16", False),
        # Training backward: float32 gradients, as the attention backward writes them, into bf16
        # activations; shared key heads and an odd length.
        _rope("norm+rope, training backward", 4, 4095, 16, 4, 128, "bf16", True),
        # One user, short context: latency.
        _decode("decode, one short sequence", 1, 32, 8, 128, "bf16", 16, 700, 700),
        # A full serving batch: 64 sequences of up to 8192 tokens, as the decode benchmark, with
        # grouped key heads and unequal lengths.
        _decode("decode, batch of 64", 64, 32, 8, 128, "bf16", 16, 4096, 8192),
        # One very long context (262144 tokens), split over the whole card.
        _decode("decode, one long sequence", 1, 32, 8, 128, "bf16", 64, 262131, 262131),
        # Streaming chat in float32: a window and four first tokens, unequal lengths from one
        # token up, a page that is no power of two, one key head per query head.
        _decode("decode, window and sinks fp32", 16, 16, 16, 64, "fp32", 24, 1, 20000, 4095, 4),
        # One user: top-k then top-p over a small vocabulary.
        _sample("sample, one row", 1, 32000, "bf16", "top_k_top_p"),
        # A wide batch with the usual top-k and top-p.
        _sample("sample, top-k and top-p", 256, 131072, "bf16", "top_k_top_p"),
        # The same batch with top-p alone: sharp rows and some flat ones, whose nucleus holds
        # thousands of tokens.
        _sample("sample, top-p alone", 256, 131072, "bf16", "top_p"),
        # Every request with its own settings (greedy, unrestricted, min-p, large top-k) on
        # float32 logits of an odd vocabulary.
        _sample("sample, mixed requests fp32", 64, 100003, "fp32", "mixed"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "decode", "decode", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16])
    heads = kv_heads * group
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
    if op == "rope":
        rows = (1 << 25) // ((heads + kv_heads) * dim)
        seq = _log_int(rng, 1, 4096)
        batch = max(1, min(_log_int(rng, 1, 64), rows // seq))
        return _rope("", batch, seq, heads, kv_heads, dim, dtype, rng.random() < 0.5,
                     rng.choice([0, 0, 17]))
    if op == "append":
        seq = rng.choice([1, 1, _log_int(rng, 2, 1500)])
        batch = max(1, min(_log_int(rng, 1, 128), 8192 // seq))
        return _append("", batch, seq, heads, kv_heads, dim, dtype, rng.choice([8, 16, 24, 64]),
                       _log_int(rng, 1, 1000), rng.random() < 0.7)
    if op == "decode":
        keys = min(1 << 29, (1 << 28) * 4 // SIZES[dtype]) // (kv_heads * max(dim, 64))
        keys = min(keys, (1 << 27) // heads)  # the plain form's scores
        top = _log_int(rng, 1, min(200000, keys))
        batch = max(1, min(_log_int(rng, 1, 256), keys // top))
        low = rng.choice([1, max(1, top // 2), top])
        window, sinks = (-1, 0) if rng.random() < 0.6 else (_log_int(rng, 1, top + 1),
                                                            rng.choice([0, 4, 37]))
        return _decode("", batch, heads, kv_heads, dim, dtype, rng.choice([1, 8, 16, 24, 64, 128]),
                       low, top, window, sinks)
    vocab = _log_int(rng, 50, 150000)
    batch = max(1, min(_log_int(rng, 1, 512), (1 << 25) // vocab))
    return _sample("", batch, vocab, dtype, rng.choice(["top_k_top_p", "top_p", "mixed"]))


# ------------------------------------------------------------------- work
def _visible(case):
    """Mean number of keys that a sequence of the case sees."""
    lo, hi, w = case["min_len"], case["max_len"], case["window"]
    lens = [lo + (hi - lo) * i // 63 for i in range(64)]
    if w < 0:
        return sum(lens) / 64.0
    return sum(min(n, w + 1) + min(case["sinks"], max(0, n - w - 1)) for n in lens) / 64.0


def work(case):
    size = SIZES[case["dtype"]]
    op = case["op"]
    if op == "rope":
        tokens = case["batch"] * case["seq"]
        values = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        tables = case["seq"] * case["dim"] * 4  # cos and sin
        # backward: float32 gradient in, activation in, gradient of the activation out
        moved = (4 + 2 * size) if case["grad"] else 2 * size
        return {"bytes": values * moved + tables, "flops": values * (20 if case["grad"] else 10)}
    if op == "append":
        # Real tokens (the mean of the rows' counts) are read and written, padding queries only
        # written.
        real = case["batch"] * (max(1, case["seq"] // 2) + case["seq"]) / 2
        padding = case["batch"] * case["seq"] - real
        rotated = real * (case["heads"] + case["kv_heads"]) * case["dim"]
        copied = real * case["kv_heads"] * case["dim"]
        zeroed = padding * case["heads"] * case["dim"]
        return {"bytes": size * (2 * rotated + 2 * copied + zeroed) + real * case["dim"] * 4,
                "flops": rotated * (10 if case["norm"] else 6)}
    if op == "decode":
        keys = case["batch"] * _visible(case)
        pairs = keys * case["heads"]
        ends = 2 * case["batch"] * case["heads"] * case["dim"] * size
        table = 4 * keys / case["page"]
        return {"bytes": 2 * keys * case["kv_heads"] * case["dim"] * size + ends + table,
                "flops": 4 * pairs * case["dim"]}
    values = case["batch"] * case["vocab"]
    return {"bytes": values * size + case["batch"] * 28, "flops": values * 4}


# ---------------------------------------------------------------- prepare
def _tables(rows, dim):
    theta = ROPE_BASE ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64) / dim)
    angles = torch.arange(rows, dtype=torch.float64)[:, None] * theta[None, :]
    return torch.cos(angles).float().cuda(), torch.sin(angles).float().cuda()


def _pages(gen, batch, most, page):
    """A block table of shuffled pages for sequences of up to `most` slots, and the page count."""
    columns = max(1, -(-most // page))
    total = batch * columns + 3
    order = torch.randperm(total, generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    return order[:batch * columns].reshape(batch, columns).contiguous(), total


def _ints(gen, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)


def _logits(gen, case):
    """Model-like logits: a broad bulk and a few dozen candidates above it, far above in most rows
    and hardly in one of eight."""
    B, V = case["batch"], case["vocab"]
    x = 2.0 * torch.randn((B, V), generator=gen, device="cuda")
    n = min(V, 64)
    at = torch.randint(0, V // n, (B, n), generator=gen, device="cuda")
    at = at + torch.arange(n, device="cuda") * (V // n)
    lift = 9.0 + 2.5 * torch.randn((B, n), generator=gen, device="cuda")
    flat = torch.rand((B, 1), generator=gen, device="cuda") < 0.125
    x.scatter_(1, at, torch.where(flat, lift * 0.5, lift + 3.0))
    return x.to(DTYPES[case["dtype"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    op = case["op"]

    def normal(*shape, dtype=dt):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    if op == "sample":
        B, V, kind = case["batch"], case["vocab"], case["kind"]
        s = {"case": case, "logits": _logits(gen, case),
             "u": torch.rand((B,), generator=gen, device="cuda")}
        full = lambda v, d=torch.float32: torch.full((B,), v, dtype=d, device="cuda")  # noqa: E731
        if kind == "top_k_top_p":
            s |= {"temperature": full(0.8), "top_k": full(50, torch.int32), "top_p": full(0.95),
                  "min_p": full(0.0)}
        elif kind == "top_p":
            s |= {"temperature": full(1.0), "top_k": full(0, torch.int32), "top_p": full(0.9),
                  "min_p": full(0.0)}
        else:
            pick = lambda *v, d=torch.float32: torch.tensor(v, dtype=d, device="cuda")[  # noqa: E731
                torch.randint(0, len(v), (B,), generator=gen, device="cuda")]
            s |= {"temperature": pick(0.0, 0.5, 0.8, 1.0, 1.3),
                  "top_k": pick(0, 0, 1, 40, 1000, 5000, d=torch.int32),
                  "top_p": pick(1.0, 1.0, 0.5, 0.9, 0.99), "min_p": pick(0.0, 0.0, 0.05, 0.2)}
        return s
    B, H, Hkv, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if op == "decode":
        lens = _ints(gen, case["min_len"], case["max_len"], B)
        table, total = _pages(gen, B, case["max_len"], case["page"])
        return {"case": case, "q": normal(B, H, D), "lens": lens, "table": table,
                "k": normal(total, Hkv, case["page"], D), "v": normal(total, Hkv, case["page"], D)}
    S = case["seq"]
    # Head views of one fused projection's output, as the layers hold them.
    qkv = normal(B, S, (H + 2 * Hkv) * D)
    s = {"case": case, "q": qkv[..., :H * D].unflatten(-1, (H, D)),
         "k": qkv[..., H * D:(H + Hkv) * D].unflatten(-1, (Hkv, D)),
         "v": qkv[..., (H + Hkv) * D:].unflatten(-1, (Hkv, D)),
         "wq": 1.0 + 0.2 * normal(D, dtype=torch.float32),
         "wk": 1.0 + 0.2 * normal(D, dtype=torch.float32)}
    if op == "append":
        start = _ints(gen, 0, case["max_start"], B)
        n_new = _ints(gen, max(1, S // 2), S, B)
        table, total = _pages(gen, B, case["max_start"] + S, case["page"])
        s |= {"start": start, "n_new": n_new, "table": table,
              "kp": torch.zeros((total, Hkv, case["page"], D), dtype=dt, device="cuda"),
              "vp": torch.zeros((total, Hkv, case["page"], D), dtype=dt, device="cuda"),
              "rope": _tables(case["max_start"] + S, D)}
        if not case["norm"]:
            s["wq"] = s["wk"] = None
        return s
    s["rope"] = _tables(case["pos0"] + S, D)
    if case["grad"]:
        s |= {"dq": normal(B, S, H, D, dtype=torch.float32),
              "dk": normal(B, S, Hkv, D, dtype=torch.float32)}
    return s


# ------------------------------------------------------------ plain forms
def _rotate(x, cos, sin):
    h = x.shape[-1] // 2
    return torch.cat([x[..., :h] * cos - x[..., h:] * sin, x[..., h:] * cos + x[..., :h] * sin], -1)


def _norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _plain_rope(s):
    c = s["case"]
    rows = slice(c["pos0"], c["pos0"] + c["seq"])
    cos, sin = s["rope"][0][rows, None], s["rope"][1][rows, None]
    return tuple(_rotate(_norm(x.float(), w), cos, sin).to(x.dtype)
                 for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])))


def _norm_grad(x, w, dy, cos, sin):
    xf = x.float()
    r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
    xh = xf * r
    dz = _rotate(dy, cos, -sin)
    g = dz * w
    dx = r * (g - xh * (g * xh).mean(-1, keepdim=True))
    return dx.to(x.dtype), (dz * xh).sum((0, 1, 2))


def _plain_rope_grad(s):
    c = s["case"]
    rows = slice(c["pos0"], c["pos0"] + c["seq"])
    cos, sin = s["rope"][0][rows, None], s["rope"][1][rows, None]
    dq, dwq = _norm_grad(s["q"], s["wq"], s["dq"], cos, sin)
    dk, dwk = _norm_grad(s["k"], s["wk"], s["dk"], cos, sin)
    return dq, dk, dwq, dwk


def _plain_append(s):
    c = s["case"]
    B, S, page = c["batch"], c["seq"], c["page"]
    step = torch.arange(S, device="cuda")[None, :]
    pos = s["start"].long()[:, None] + step
    cos, sin = s["rope"][0][pos][:, :, None], s["rope"][1][pos][:, :, None]
    q, k = s["q"].float(), s["k"].float()
    if s["wq"] is not None:
        q, k = _norm(q, s["wq"]), _norm(k, s["wk"])
    q, k = _rotate(q, cos, sin).to(s["q"].dtype), _rotate(k, cos, sin).to(s["k"].dtype)
    real = (step < s["n_new"].long()[:, None]).reshape(-1)
    at = torch.gather(s["table"].long(), 1, pos // page).reshape(-1)[real]
    off = (pos % page).reshape(-1)[real]
    s["kp"][at, :, off] = k.reshape(B * S, *k.shape[2:])[real]
    s["vp"][at, :, off] = s["v"].reshape(B * S, *k.shape[2:])[real]
    # queries past a row's new tokens are padding
    return torch.where(real.reshape(B, S, 1, 1), q, torch.zeros_like(q)), s["kp"], s["vp"]


def _plain_decode(s):
    c = s["case"]
    B, H, Hkv, D = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    table = s["table"].long()
    n = table.shape[1] * c["page"]
    k = s["k"][table].permute(0, 2, 1, 3, 4).reshape(B, Hkv, n, D).float()
    scores = torch.matmul(s["q"].float().reshape(B, Hkv, H // Hkv, D), k.transpose(2, 3))
    scores = scores.reshape(B, H, n) * (1.0 / math.sqrt(D))
    del k
    j = torch.arange(n, device="cuda")[None, :]
    last = s["lens"].long()[:, None] - 1
    seen = j <= last
    if c["window"] >= 0:
        seen = seen & ((j >= last - c["window"]) | (j < c["sinks"]))
    scores = torch.where(seen[:, None], scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    v = s["v"][table].permute(0, 2, 1, 3, 4).reshape(B, Hkv, n, D).float()
    out = torch.matmul(p.reshape(B, Hkv, H // Hkv, n), v).reshape(B, H, D) / total
    return out.to(s["q"].dtype), (top + torch.log(total)).reshape(B, H)


def _share(total, part):
    """floor(total * part / 2^24) of whole numbers, without leaving 64 bits."""
    return (total >> 24) * part + (((total & 0xFFFFFF) * part) >> 24)


def _plain_sample(s):
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top = x.amax(-1, keepdim=True)
    t = s["temperature"][:, None]
    inv = 1.0 / torch.where(t > 0, t, torch.ones_like(t))
    w = torch.exp(torch.where(x == top, torch.zeros_like(x), (x - top) * inv))
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    ws = torch.gather(w, 1, order)
    qs = (ws * WEIGHT_ONE).to(torch.int64)
    rank = torch.arange(x.shape[1], device=x.device)[None, :]
    k = s["top_k"].long()[:, None]
    qs = torch.where((rank < k) | (k <= 0), qs, torch.zeros_like(qs))
    before = torch.cumsum(qs, -1) - qs
    part = (s["top_p"].clamp(0, 1) * 16777216.0).to(torch.int64)[:, None]
    bound = _share(qs.sum(-1, keepdim=True), part)
    keep = ((before < bound) | (rank == 0)) & (ws >= s["min_p"][:, None])
    kept = torch.zeros_like(qs).scatter_(1, order, torch.where(keep, qs, torch.zeros_like(qs)))
    run_sum = torch.cumsum(kept, -1)
    u = (s["u"] * 16777216.0).to(torch.int64).clamp(0, 16777215)[:, None]
    token = (run_sum <= _share(run_sum[:, -1:], u)).sum(-1)
    return torch.where(s["temperature"] > 0, token, order[:, 0])


def run(state):
    c = state["case"]
    op = c["op"]
    if not own:
        if op == "rope":
            return _plain_rope_grad(state) if c["grad"] else _plain_rope(state)
        return {"append": _plain_append, "decode": _plain_decode, "sample": _plain_sample}[op](state)
    from enilnets_b200 import kernels
    if op == "rope":
        if c["grad"]:
            return kernels.qk_norm_rope_backward(
                state["dq"], state["dk"], state["q"], state["k"], state["wq"], state["wk"],
                eps=EPS, rope=state["rope"], pos0=c["pos0"])
        return kernels.qk_norm_rope(state["q"], state["k"], state["wq"], state["wk"], eps=EPS,
                                    rope=state["rope"], pos0=c["pos0"])
    if op == "append":
        q = kernels.qk_norm_rope_append(
            state["q"], state["k"], state["v"], state["kp"], state["vp"], state["table"],
            state["start"], n_new=state["n_new"], q_weight=state["wq"], k_weight=state["wk"],
            eps=EPS, rope=state["rope"])
        return q, state["kp"], state["vp"]
    if op == "decode":
        return kernels.attention_decode_paged(
            state["q"], state["k"], state["v"], state["table"], state["lens"],
            window=None if c["window"] < 0 else c["window"], sinks=c["sinks"],
            out_dtype=state["q"].dtype, return_lse=True)
    return kernels.sample_tokens(state["logits"], state["u"], temperature=state["temperature"],
                                 top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])


# ------------------------------------------------------------------ exact
def _turn64(x, pos, dim, back=False):
    """x (..., heads, dim) as complex numbers turned by each position's angles."""
    theta = ROPE_BASE ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64) / dim)
    angle = pos.double()[..., None] * theta.cuda()
    # the tables are 32-bit inputs of the operator
    turn = torch.complex(torch.cos(angle).float().double(), torch.sin(angle).float().double())
    turn = (turn.conj() if back else turn).unsqueeze(-2)
    z = torch.complex(x[..., :dim // 2].contiguous(), x[..., dim // 2:].contiguous()) * turn
    return torch.cat([z.real, z.imag], -1)


def _unit64(x):
    x = x.double()
    return x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        tokens = []
        rows = s["logits"].double().cpu()
        for b in range(case["batch"]):
            t = float(s["temperature"][b])
            if t == 0:
                tokens.append(int(rows[b].argmax()))
                continue
            p = torch.softmax(rows[b] / t, -1)
            v, i = torch.sort(rows[b], descending=True, stable=True)
            p = p[i]
            k = int(s["top_k"][b])
            if k > 0:
                p[k:] = 0
            p = p / p.sum()
            p[torch.cumsum(p, 0) - p >= float(s["top_p"][b])] = 0
            p[p < float(s["min_p"][b]) * p[0]] = 0
            c = torch.cumsum(torch.zeros_like(p).scatter_(0, i, p), 0)
            tokens.append(int((c <= float(s["u"][b]) * c[-1]).sum()))
        return torch.tensor(tokens)
    D = case["dim"]
    if op == "decode":
        outs, lses = [], []
        for b in range(case["batch"]):
            n = int(s["lens"][b])
            j = torch.arange(n, device="cuda")
            if case["window"] >= 0:
                j = j[(j > n - 2 - case["window"]) | (j < case["sinks"])]
            page, off = s["table"][b].long()[j // case["page"]], j % case["page"]
            for h in range(case["kv_heads"]):
                g = case["heads"] // case["kv_heads"]
                k, v = s["k"][page, h, off].double(), s["v"][page, h, off].double()
                a = s["q"][b, h * g:(h + 1) * g].double() @ k.T / math.sqrt(D)
                outs.append(torch.softmax(a, -1) @ v)
                lses.append(torch.logsumexp(a, -1))
        shape = (case["batch"], case["heads"])
        return torch.cat(outs).reshape(*shape, D), torch.cat(lses).reshape(shape)
    B, S = case["batch"], case["seq"]
    if op == "append":
        pos = s["start"].double()[:, None] + torch.arange(S, device="cuda")
        q, k = s["q"].double(), s["k"].double()
        if case["norm"]:
            q, k = _unit64(q) * s["wq"].double(), _unit64(k) * s["wk"].double()
        q, k = _turn64(q, pos, D), _turn64(k, pos, D)
        kp, vp = s["kp"].double(), s["vp"].double()
        for b in range(B):
            n, first = int(s["n_new"][b]), int(s["start"][b])
            q[b, n:] = 0
            at = torch.arange(first, first + n, device="cuda")
            page, off = s["table"][b].long()[at // case["page"]], at % case["page"]
            kp[page, :, off] = k[b, :n]
            vp[page, :, off] = s["v"][b, :n].double()
        return q, kp, vp
    pos = torch.arange(case["pos0"], case["pos0"] + S, device="cuda")
    if not case["grad"]:
        return (_turn64(_unit64(s["q"]) * s["wq"].double(), pos, D),
                _turn64(_unit64(s["k"]) * s["wk"].double(), pos, D))
    got = []
    for x, w, dy in ((s["q"], s["wq"], s["dq"]), (s["k"], s["wk"], s["dk"])):
        dz = _turn64(dy.double(), pos, D, back=True)
        u = _unit64(x)
        n = torch.sqrt(x.double().pow(2).sum(-1, keepdim=True) / D + EPS)
        g = dz * w.double()
        got.append(((g - u * (g * u).sum(-1, keepdim=True) / D) / n, (dz * u).flatten(0, 2).sum(0)))
    return got[0][0], got[1][0], got[0][1], got[1][1]
