"""What the performance of the attention operators (`rocshmem_b200.ops.attention`) is measured on.

Kinds of cases:

* ``rope``    RMS norm of every query and key head with the position rotation in the same pass; ``train``: with the
              gradients of queries, keys and both norm weights;
* ``write``   keys and values of new tokens into a paged cache, in 16 bits or quantised to e4m3 on the way;
* ``read``    tokens of a paged cache read back;
* ``attend``  attention of one new token for each sequence over a paged cache;
* ``join``    partial results of several parts of a cache (those of the PEs that hold it) joined into one.

``run`` computes a case in plain torch in 32 bits, or, with ``own``, through the framework's operators.
"""
from __future__ import annotations

import types

import torch

own = False

EPS = 1e-6
E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": E4M3}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}


def listed():
    """The listed cases."""
    return [
        # One decode step's projections of 64 sequences, views of one fused buffer: latency.
        {"name": "rope_decode", "kind": "rope", "tokens": 64, "pad": 0, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "dtype": "bf16", "weight": "bf16", "interleaved": False, "fused": True, "train": False,
         "positions": 131072},
        # A training micro-batch, forward and backward.
        {"name": "rope_train", "kind": "rope", "tokens": 16384, "pad": 0, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "dtype": "bf16", "weight": "fp32", "interleaved": False, "fused": False, "train": True,
         "positions": 16384},
        # The new tokens of a decode step, quantised into the cache; three rows of the batch are padding.
        {"name": "write_e4m3_decode", "kind": "write", "tokens": 64, "pad": 3, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "bf16", "cache": "e4m3", "fused": True},
        # A long prompt, quantised as it is written.
        {"name": "write_e4m3_prefill", "kind": "write", "tokens": 32768, "pad": 0, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "cache": "e4m3", "fused": True},
        # A prefix of an odd length read back in order to continue a prompt.
        {"name": "read_e4m3_prefix", "kind": "read", "tokens": 16381, "pad": 0, "kv_heads": 8, "dim": 128, "page": 16,
         "dtype": "bf16", "cache": "e4m3"},
        # A short prefix of a small model.
        {"name": "read_fp16_short", "kind": "read", "tokens": 300, "pad": 0, "kv_heads": 4, "dim": 64, "page": 32,
         "dtype": "fp16", "cache": "fp16"},
        # Four short conversations: latency.
        {"name": "attend_small", "kind": "attend", "batch": 4, "longest": 300, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "dtype": "bf16", "cache": "bf16", "softcap": 0.0, "window": 0},
        # An ordinary batch of ragged lengths.
        {"name": "attend_batch", "kind": "attend", "batch": 64, "longest": 4096, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "dtype": "bf16", "cache": "bf16", "softcap": 0.0, "window": 0},
        # Two very long documents in a quantised cache.
        {"name": "attend_e4m3_long", "kind": "attend", "batch": 2, "longest": 524287, "heads": 64, "kv_heads": 8,
         "dim": 128, "page": 64, "dtype": "bf16", "cache": "e4m3", "softcap": 0.0, "window": 0},
        # A layer with capped scores and a sliding window, five query heads to a key head.
        {"name": "attend_window_cap", "kind": "attend", "batch": 96, "longest": 8192, "heads": 40, "kv_heads": 8,
         "dim": 64, "page": 32, "dtype": "fp16", "cache": "fp16", "softcap": 50.0, "window": 2048},
        # The halves of a small batch's caches on two PEs.
        {"name": "join_2", "kind": "join", "parts": 2, "batch": 16, "heads": 32, "dim": 128, "dtype": "bf16"},
        # A large batch over eight PEs.
        {"name": "join_8", "kind": "join", "parts": 8, "batch": 512, "heads": 64, "dim": 128, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case of the ranges that the listed ones stand for."""
    kind = rng.choice(["rope", "rope", "write", "read", "attend", "attend", "attend", "join"])
    dim = rng.choice([64, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 12, 16, 24])
    if kind == "rope":
        train = rng.random() < 0.5
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = max(1, 80_000_000 // ((heads + kv_heads) * dim * (2 if dtype == "fp32" else 1)))
        tokens = _log(rng, 1, min(32768, most))
        return {"kind": "rope", "tokens": tokens, "pad": rng.choice([0, 0, min(3, tokens - 1)]), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2]), "dtype": dtype,
                "weight": rng.choice([dtype, "fp32"]), "interleaved": rng.random() < 0.3,
                "fused": rng.random() < 0.6, "train": train, "positions": rng.choice([32768, 131072])}
    if kind in ("write", "read"):
        dtype = rng.choice(["bf16", "fp16"])
        tokens = _log(rng, 1, max(1, min(65536, 32_000_000 // (kv_heads * dim))))
        c = {"kind": kind, "tokens": tokens, "pad": rng.choice([0, 0, min(5, tokens - 1)]), "kv_heads": kv_heads,
             "dim": dim, "page": rng.choice([16, 32, 64, 128]), "dtype": dtype, "cache": rng.choice(["e4m3", dtype])}
        return dict(c, fused=rng.random() < 0.6) if kind == "write" else c
    if kind == "attend":
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        cache = rng.choice(["e4m3", dtype])
        batch = _log(rng, 1, 256)
        most = 250_000_000 // (batch * kv_heads * dim * SIZES[cache])
        return {"kind": "attend", "batch": batch, "longest": _log(rng, 1, max(1, min(524288, most))),
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128]),
                "dtype": dtype, "cache": cache, "softcap": rng.choice([0.0, 0.0, 30.0]),
                "window": rng.choice([0, 0, 0, 1000])}
    parts, batch = rng.randint(2, 16), _log(rng, 1, 512)
    most = max(1, 33_000_000 // (parts * batch * dim))
    return {"kind": "join", "parts": parts, "batch": batch, "heads": min(heads, most), "dim": dim,
            "dtype": rng.choice(["bf16", "fp16", "fp32"])}


# ---- inputs ---------------------------------------------------------------------------------------------------

def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _heads(g, tokens, counts, dim, dtype, fused):
    """Tensors [tokens, count, dim], one for each of `counts`: views of one buffer, or each on its own."""
    if not fused:
        return [_randn(g, tokens, n, dim, dtype=dtype) for n in counts]
    both = _randn(g, tokens, sum(counts), dim, dtype=dtype)
    return list(both.split(counts, dim=1))


def _cache(g, pages, case):
    """A cache's four tensors with content: `k`, `v` [pages, kv_heads, page, dim], for e4m3 with one factor a row."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    if case["cache"] != "e4m3":
        dtype = TYPES[case["cache"]]
        return _randn(g, *shape, dtype=dtype), _randn(g, *shape, dtype=dtype), None, None
    k, v = (_randn(g, *shape, scale=150.0).clamp_(-448, 448).to(E4M3) for _ in range(2))
    ks, vs = ((torch.rand(shape[:3], generator=g, device="cuda") + 0.5) / 150.0 for _ in range(2))
    return k, v, ks, vs


def prepare(case, seed):
    """Inputs made from the seed."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = types.SimpleNamespace(case=case)
    kind, dtype = case["kind"], TYPES[case["dtype"]]
    if kind == "rope":
        T, D, R = case["tokens"], case["dim"], case["rotary"]
        counts = [case["heads"], case["kv_heads"]]
        fused = case["fused"]
        s.q, s.k = _heads(g, T, counts + [case["kv_heads"]], D, dtype, True)[:2] if fused else \
            _heads(g, T, counts, D, dtype, False)
        wt = TYPES[case["weight"]]
        s.q_weight, s.k_weight = (_randn(g, D, scale=0.2).add_(1.0).to(wt) for _ in range(2))
        # Tokens of packed sequences: each starts at a position of its own and counts on from there.
        start = torch.randint(0, case["positions"] // 2, (T,), generator=g, device="cuda")
        step = torch.arange(T, device="cuda")
        length = 4096
        s.positions = ((start[step // length * length] + step % length) % case["positions"]).to(torch.int32)
        s.positions[T - case["pad"]:] = -1
        inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
        angle = torch.arange(case["positions"], dtype=torch.float64, device="cuda")[:, None] * inv
        s.table = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        if case["train"]:
            s.q, s.k = s.q.detach().requires_grad_(), s.k.detach().requires_grad_()
            s.q_weight.requires_grad_()
            s.k_weight.requires_grad_()
            s.gq, s.gk = _heads(g, T, counts, D, dtype, False)
    elif kind in ("write", "read"):
        T, pad, P = case["tokens"], case["pad"], case["page"]
        pages = (T + P - 1) // P + 3
        s.k_cache, s.v_cache, s.k_scale, s.v_scale = _cache(g, pages, case)
        # Consecutive tokens fill pages that lie anywhere in the cache; the first page is begun in its middle.
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(T, device="cuda") + P // 2
        s.slots = order[at // P] * P + at % P
        s.slots[T - pad:] = -1
        if kind == "write":
            s.k, s.v = _heads(g, T, [case["kv_heads"]] * 2, case["dim"], dtype, case["fused"])
    elif kind == "attend":
        B, P, longest = case["batch"], case["page"], case["longest"]
        # Lengths between a quarter of the longest and the longest, which one sequence has.
        s.lengths = (longest - torch.randint(0, longest - longest // 4, (B,), generator=g, device="cuda")).to(torch.int32)
        s.lengths[B // 2] = longest
        per = (longest + P - 1) // P
        pages = B * per
        s.k_cache, s.v_cache, s.k_scale, s.v_scale = _cache(g, pages, case)
        s.block_table = torch.randperm(pages, generator=g, device="cuda").view(B, per).to(torch.int32)
        used = torch.arange(per, device="cuda")[None] * P < s.lengths[:, None]
        s.block_table = torch.where(used, s.block_table, -1).contiguous()
        s.q = _randn(g, B, case["heads"], case["dim"], dtype=dtype, scale=1.5)
    else:
        n, B, H, D = case["parts"], case["batch"], case["heads"], case["dim"]
        s.outs = _randn(g, n, B, H, D)
        s.lses = _randn(g, n, B, H, scale=2.0)
        # A sequence may have no tokens on some of the PEs.
        s.lses[torch.rand((n, B, H), generator=g, device="cuda") < 0.05] = float("-inf")
    torch.cuda.synchronize()
    return s


# ---- the operators in plain torch ---------------------------------------------------------------------------------

def _rotate(y, c, s, interleaved):
    """Pairs of the last dimension of `y` rotated by the angles whose cosines and sines are `c` and `s`."""
    if interleaved:
        a, b = y[..., 0::2], y[..., 1::2]
        return torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    a, b = y.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _norm_rope(x, weight, positions, table, interleaved):
    R = table.shape[1]
    xf = x.float()
    y = xf * torch.rsqrt((xf * xf).mean(dim=-1, keepdim=True) + EPS) * weight.float()
    angles = table[positions.clamp(min=0)][:, None, :]
    c, s = angles[..., :R // 2], angles[..., R // 2:]
    y = torch.cat([_rotate(y[..., :R], c, s, interleaved), y[..., R:]], dim=-1)
    return torch.where((positions >= 0)[:, None, None], y, 0.0).to(x.dtype)


def _plain_write(s):
    T, P = s.case["tokens"] - s.case["pad"], s.case["page"]
    page, offset = s.slots[:T] // P, s.slots[:T] % P
    for_each = ((s.k, s.k_cache, s.k_scale), (s.v, s.v_cache, s.v_scale))
    (xk, ck, sk), (xv, cv, sv) = for_each

    def put(x, cache, scale):
        x = x[:T].float()
        if scale is None:
            cache[page, :, offset] = x.to(cache.dtype)
            return
        most = x.abs().amax(dim=-1).clamp(min=2.0 ** -110)
        codes = (x * (448.0 / most)[..., None]).clamp(-448, 448).to(E4M3)
        cache.view(torch.uint8)[page, :, offset] = codes.view(torch.uint8)
        scale[page, :, offset] = most * (1.0 / 448.0)

    put(xk, ck, sk)
    put(xv, cv, sv)


def _plain_rows(s, cache, scale):
    """Rows of the cache by slot, in 32 bits; zeros for padding."""
    P = s.case["page"]
    at = s.slots.clamp(min=0)
    raw = cache.view(torch.uint8)[at // P, :, at % P].view(E4M3) if scale is not None else cache[at // P, :, at % P]
    x = raw.float()
    if scale is not None:
        x = x * scale[at // P, :, at % P][..., None]
    return torch.where((s.slots >= 0)[:, None, None], x, 0.0).to(TYPES[s.case["dtype"]])


def _plain_sequences(s, cache, scale):
    """The sequences' rows in order, [batch, kv_heads, longest, dim] in 32 bits."""
    table = s.block_table.clamp(min=0).long()
    B, per = table.shape
    raw = cache.view(torch.uint8)[table].view(E4M3) if scale is not None else cache[table]
    x = raw.float()
    if scale is not None:
        x = x * scale[table][..., None]
    return x.transpose(1, 2).reshape(B, s.case["kv_heads"], per * s.case["page"], s.case["dim"])


def _plain_attend(s):
    case = s.case
    B, H, K, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    keys = _plain_sequences(s, s.k_cache, s.k_scale)
    q = s.q.float().view(B, K, H // K, D)
    scores = (q @ keys.transpose(-1, -2)) * D ** -0.5
    del keys
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    at = torch.arange(scores.shape[-1], device=scores.device)[None]
    n = s.lengths[:, None]
    seen = at < n
    if case["window"]:
        seen = seen & (at >= n - case["window"])
    scores = torch.where(seen[:, None, None], scores, float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - top)
    total = p.sum(dim=-1, keepdim=True)
    out = ((p / total) @ _plain_sequences(s, s.v_cache, s.v_scale)).view(B, H, D).to(s.q.dtype)
    return {"out": out, "lse": (top + total.log()).view(B, H)}


def _plain_join(s):
    top = s.lses.amax(dim=0)
    w = torch.exp(s.lses - torch.where(top > float("-inf"), top, 0.0))
    total = w.sum(dim=0)
    out = (s.outs * w[..., None]).sum(dim=0) / torch.where(total > 0, total, 1.0)[..., None]
    return {"out": out.to(TYPES[s.case["dtype"]]), "lse": top + torch.where(total > 0, total, 1.0).log()}


def run(s):
    """One pass."""
    case = s.case
    kind = case["kind"]
    if own:
        from rocshmem_b200.ops import attention
    if kind == "rope":
        if own:
            q, k = attention.qk_norm_rope(s.q, s.k, s.q_weight, s.k_weight, s.positions, s.table, eps=EPS,
                                          interleaved=case["interleaved"])
        else:
            q, k = (_norm_rope(x, w, s.positions, s.table, case["interleaved"])
                    for x, w in ((s.q, s.q_weight), (s.k, s.k_weight)))
        if not case["train"]:
            return {"q": q, "k": k}
        gq, gk, gwq, gwk = torch.autograd.grad((q, k), (s.q, s.k, s.q_weight, s.k_weight), (s.gq, s.gk))
        return {"q": q.detach(), "k": k.detach(), "gq": gq, "gk": gk, "gwq": gwq, "gwk": gwk}
    if kind == "join":
        if own:
            out, lse = attention.attention_join(s.outs, s.lses, dtype=TYPES[case["dtype"]])
            return {"out": out, "lse": lse}
        return _plain_join(s)
    cache = attention.KvCache(s.k_cache, s.v_cache, s.k_scale, s.v_scale) if own else None
    if kind == "write":
        if own:
            attention.kv_cache_write(cache, s.k, s.v, s.slots)
        else:
            _plain_write(s)
        return [x for x in (s.k_cache, s.v_cache, s.k_scale, s.v_scale) if x is not None]
    if kind == "read":
        if own:
            return attention.kv_cache_read(cache, s.slots, dtype=TYPES[case["dtype"]])
        return _plain_rows(s, s.k_cache, s.k_scale), _plain_rows(s, s.v_cache, s.v_scale)
    if own:
        out, lse = attention.paged_attention(s.q, cache, s.block_table, s.lengths, softcap=case["softcap"],
                                             window=case["window"], return_lse=True)
        return {"out": out, "lse": lse}
    return _plain_attend(s)


def work(case):
    """Bytes that a pass has to read and write, each once, and its floating-point operations."""
    kind, size = case["kind"], SIZES[case["dtype"]]
    D = case["dim"]
    if kind == "rope":
        T, n = case["tokens"], case["tokens"] * (case["heads"] + case["kv_heads"]) * D
        table = 4 * case["rotary"] * min(T, case["positions"]) + 4 * T
        if not case["train"]:
            return {"bytes": 2 * n * size + table, "flops": 9.0 * n}
        return {"bytes": 5 * n * size + 2 * table, "flops": 26.0 * n}
    if kind in ("write", "read"):
        rows = 2 * (case["tokens"] - case["pad"]) * case["kv_heads"]
        row = D * (size + SIZES[case["cache"]]) + (4 if case["cache"] == "e4m3" else 0)
        return {"bytes": rows * row + 8 * case["tokens"], "flops": 2.0 * rows * D}
    if kind == "join":
        rows = case["batch"] * case["heads"]
        return {"bytes": rows * (case["parts"] * (4 * D + 4) + D * size + 4), "flops": 2.0 * rows * case["parts"] * D}
    # Lengths are spread evenly between a quarter of the longest and the longest, which one sequence has.
    lo, hi, w = case["longest"] // 4 + 1, case["longest"], case["window"]
    mean = (lo + hi) / 2.0 if not w or w >= hi else sum(min(w, n) for n in range(lo, hi + 1)) / (hi - lo + 1.0)
    tokens = (case["batch"] - 1) * mean + (min(w, hi) if w else hi)
    row = D * SIZES[case["cache"]] + (4 if case["cache"] == "e4m3" else 0)
    H, B = case["heads"], case["batch"]
    return {"bytes": 2 * tokens * case["kv_heads"] * row + B * H * (2 * D * size + 4) + 4 * tokens / case["page"],
            "flops": 4.0 * tokens * H * D}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------

def _exact_rope(s, x, weight, grad):
    """Output, and for `grad` the gradients of the input and the weight, one pair of elements after the other rule."""
    case = s.case
    D, R = case["dim"], case["rotary"]
    x, w = x.detach().double(), weight.detach().double()
    first = torch.arange(R // 2, device=x.device) * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else R // 2)
    live = (s.positions >= 0).double()[:, None, None]
    angles = s.table.double()[s.positions.clamp(min=0).long()]
    cos, sin = angles[:, None, :R // 2], angles[:, None, R // 2:]
    r = (x.pow(2).sum(-1, keepdim=True) / D + EPS).pow(-0.5)
    n = x * r
    y = n * w
    out = y.clone()
    out[..., first] = y[..., first] * cos - y[..., second] * sin
    out[..., second] = y[..., second] * cos + y[..., first] * sin
    out = out * live
    if grad is None:
        return out, None, None
    g = grad.double() * live
    back = g.clone()
    back[..., first] = g[..., first] * cos + g[..., second] * sin
    back[..., second] = g[..., second] * cos - g[..., first] * sin
    a = back * w
    return out, r * (a - n * ((a * n).sum(-1, keepdim=True) / D)), (back * n).sum(dim=(0, 1))


def exact(case, seed):
    """What `run` returns for these inputs, in 64 bits."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        gq, gk = (s.gq, s.gk) if case["train"] else (None, None)
        q, dq, dwq = _exact_rope(s, s.q, s.q_weight, gq)
        k, dk, dwk = _exact_rope(s, s.k, s.k_weight, gk)
        return {"q": q, "k": k, "gq": dq, "gk": dk, "gwq": dwq, "gwk": dwk} if case["train"] else {"q": q, "k": k}
    if kind == "join":
        w = s.lses.double().exp()
        total = w.sum(0)
        out = torch.einsum("nbh,nbhd->bhd", w, s.outs.double()) / total.clamp(min=1e-300)[..., None]
        return {"out": out, "lse": total.log()}
    P = case["page"]
    if kind == "write":
        got = []
        for x, cache, scale in ((s.k, s.k_cache, s.k_scale), (s.v, s.v_cache, s.v_scale)):
            flat = cache.float().double().transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
            n = case["tokens"] - case["pad"]
            x = x[:n].double()
            if scale is None:
                flat[s.slots[:n]] = x
                got.append((flat, None))
                continue
            factor = x.abs().amax(-1) / 448
            flat[s.slots[:n]] = x / factor[..., None]
            rows = scale.double().transpose(1, 2).reshape(-1, case["kv_heads"])
            rows[s.slots[:n]] = factor
            got.append((flat, rows.view(-1, P, case["kv_heads"]).transpose(1, 2)))
        values = [f.view(-1, P, case["kv_heads"], case["dim"]).transpose(1, 2) for f, _ in got]
        return values + [r for _, r in got if r is not None]

    def whole(cache, scale, pages):
        """The rows of `pages` in order, [kv_heads, rows, dim]."""
        if scale is None:
            x = cache[pages].double()
        else:
            x = cache.view(torch.uint8)[pages].view(E4M3).float().double() * scale[pages].double()[..., None]
        return x.transpose(0, 1).flatten(1, 2)

    if kind == "read":
        pages = torch.arange(s.k_cache.shape[0], device="cuda")
        got = []
        for cache, scale in ((s.k_cache, s.k_scale), (s.v_cache, s.v_scale)):
            rows = whole(cache, scale, pages)[:, s.slots.clamp(min=0)].transpose(0, 1).clone()
            rows[s.slots < 0] = 0.0
            got.append(rows)
        return tuple(got)
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    out = torch.empty((case["batch"], H, D), dtype=torch.float64, device="cuda")
    lse = torch.empty((case["batch"], H), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s.lengths.tolist()):
        lo = max(0, n - case["window"]) if case["window"] else 0
        pages = s.block_table[b, :(n + P - 1) // P].long()
        k = whole(s.k_cache, s.k_scale, pages)[:, lo:n]
        v = whole(s.v_cache, s.v_scale, pages)[:, lo:n]
        x = torch.einsum("kgd,knd->kgn", s.q[b].double().view(K, H // K, D), k) / D ** 0.5
        if case["softcap"]:
            x = case["softcap"] * torch.tanh(x / case["softcap"])
        lse[b] = torch.logsumexp(x, dim=-1).view(H)
        out[b] = torch.einsum("kgn,knd->kgd", torch.softmax(x, dim=-1), v).reshape(H, D)
    return {"out": out, "lse": lse}
