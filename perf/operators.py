"""The operators of a serving step around the quantized projections, with their
plain forms: what each computes, stated once in elementary torch operations,
and the sizes at which they are timed.

* ``plan``   ``kq.paged_plan``: block tables, token slots and positions of a
  step, built on the GPU from the requests' lengths and a list of free pages.
* ``rope``   ``kq.rope_kv_write``: rotary embedding of the new queries and
  keys, keys and values stored into their slots of a paged cache.
* ``attn``   ``kq.paged_attention``: the new tokens of every request against
  its pages (a single token, or a chunk with its causal boundary).
* ``route``  ``kq.moe_route``: experts and weights of each token from router
  logits (softmax or sigmoid scores, balance bias, groups, top-k).

A case is a dict of plain values; its request lengths are drawn from the case
itself, so that its work is known, and its tensors from the seed.
"""
import math
import random

import torch

own = False  # True: run() calls the framework's operators instead of the plain forms

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
INF = float("inf")


# --------------------------------------------------------------------------
# cases


def listed():
    return [
        # one decode step of a full batch: 64 requests take a token each, a few start a page
        {"name": "plan_decode_64", "op": "plan", "batch": 64, "q_max": 1, "ctx_max": 8192, "page": 16},
        # a long admission: 1000 requests, prompts of up to 128 tokens beside running ones
        {"name": "plan_mixed_1000", "op": "plan", "batch": 1000, "q_max": 128, "ctx_max": 3000, "page": 32},
        # a single decoding user at the Llama-3-8B attention geometry (4096 = 32 x 128, 1024 = 8 x 128)
        {"name": "rope_token", "op": "rope", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "page": 16, "dtype": "bf16", "interleaved": True},
        # a prefill chunk of 8192 tokens (the largest prefill batch of the benchmark), half-split pairs
        {"name": "rope_8192", "op": "rope", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "page": 64, "dtype": "bf16", "interleaved": False},
        # the next token of one user at a context of a thousand: latency
        {"name": "attn_token", "op": "attn", "batch": 1, "q_max": 1, "ctx_max": 999, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "softcap": 0.0, "dtype": "bf16", "lse": False},
        # the next token of 64 users, contexts of up to 16384: HBM bandwidth
        {"name": "attn_decode_64", "op": "attn", "batch": 64, "q_max": 1, "ctx_max": 16384, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "softcap": 0.0, "dtype": "bf16", "lse": False},
        # a prompt of 512 tokens with nothing cached
        {"name": "attn_prompt_512", "op": "attn", "batch": 1, "q_max": 512, "ctx_max": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "softcap": 0.0, "dtype": "bf16", "lse": False},
        # chunked prefill deep in a long document: 4096 new tokens on 32768 cached ones
        {"name": "attn_chunk_4096", "op": "attn", "batch": 1, "q_max": 4096, "ctx_max": 32768, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "softcap": 0.0, "dtype": "bf16", "lse": False},
        # decoding requests and short chunks in one batch, sliding window and capped scores, ragged sizes
        {"name": "attn_mixed_24", "op": "attn", "batch": 24, "q_max": 301, "ctx_max": 2500, "heads": 40, "kv_heads": 8,
         "dim": 64, "page": 32, "window": 1000, "softcap": 50.0, "dtype": "f16", "lse": True},
        # one token's 8 of 128 experts (Qwen3-30B-A3B-like layer)
        {"name": "route_token", "op": "route", "tokens": 1, "experts": 128, "k": 8, "scoring": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "norm": True, "scale": 1.0, "dtype": "f32"},
        # a decode batch's 8 of 256 experts, 4 of 8 groups, balance bias (DeepSeek-V3-like layer)
        {"name": "route_64_grouped", "op": "route", "tokens": 64, "experts": 256, "k": 8, "scoring": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "norm": True, "scale": 2.5, "dtype": "f32"},
        # the same layer over a prefill batch, logits in the activation type (many equal scores)
        {"name": "route_8192_grouped", "op": "route", "tokens": 8192, "experts": 256, "k": 8, "scoring": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "norm": True, "scale": 2.5, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "rope", "attn", "attn", "attn", "route"])
    if op == "plan":
        b, q = _log(rng, 1, 1200), rng.choice([1, _log(rng, 2, 512)])
        while b * q > 150_000:
            q = max(1, q // 2)
        return {"op": "plan", "batch": b, "q_max": q, "ctx_max": _log(rng, 1, 8192),
                "page": rng.choice([1, 8, 16, 24, 32, 64, 128])}
    if op == "rope":
        kv = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 128, 128, 256])
        return {"op": "rope", "tokens": _log(rng, 1, 8192), "heads": kv * rng.choice([1, 3, 4, 5, 8]), "kv_heads": kv,
                "dim": dim, "rot": rng.choice([dim, dim, dim // 2]), "page": rng.choice([1, 16, 24, 64]),
                "dtype": rng.choice(["bf16", "f16"]), "interleaved": rng.random() < 0.5}
    if op == "attn":
        b, kv = _log(rng, 1, 64), rng.choice([1, 2, 4, 8])
        q = rng.choice([1, _log(rng, 2, 16), _log(rng, 17, 2048)])
        c = {"op": "attn", "batch": b, "q_max": q, "ctx_max": rng.choice([0, _log(rng, 1, 32768)]),
             "heads": kv * rng.choice([1, 2, 3, 4, 5, 7, 8]), "kv_heads": kv, "dim": rng.choice([64, 128, 128, 256]),
             "page": rng.choice([8, 16, 16, 24, 32, 64, 128]), "window": rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
             "softcap": rng.choice([0.0, 0.0, 0.0, 30.0]), "dtype": rng.choice(["bf16", "bf16", "f16"]),
             "lse": rng.random() < 0.25}
        # the plain form holds every score of the padded batch, and the cache in 32 bits
        while (c["batch"] * c["heads"] * c["q_max"] * (c["ctx_max"] + c["q_max"]) > 1.5e9
               or c["batch"] * (c["ctx_max"] + c["q_max"]) * kv * c["dim"] > 5e8):
            big = max(("batch", "ctx_max", "q_max"), key=lambda n: c[n] * (16 if n == "batch" else 1))
            c[big] = c[big] * 3 // 4
        return c
    e = rng.choice([8, 16, 60, 64, 100, 128, 160, 256, 256, 384, 512])
    g = rng.choice([n for n in (1, 1, 2, 4, 8) if e % n == 0 and e // n >= 4])
    tg = rng.randint(1, g)
    return {"op": "route", "tokens": _log(rng, 1, 8192), "experts": e, "k": rng.randint(1, min(10, tg * (e // g))),
            "scoring": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": g, "top_groups": tg,
            "norm": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5]), "dtype": rng.choice(["f32", "bf16", "f16"])}


def _lens(case):
    """(tokens cached, new tokens) of each request, from the case alone.  The
    first request has the largest of both; in a batch of chunks a third of the
    others decode one token, and one has none."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    b, q_max, ctx_max = case["batch"], case["q_max"], case["ctx_max"]
    ctx = [ctx_max] + [rng.randint(0, ctx_max) for _ in range(b - 1)]
    q = [q_max] + [1 if rng.random() < 0.33 else rng.randint(1, q_max) for _ in range(b - 1)]
    if b >= 8 and q_max > 1:
        q[5] = 0
    return ctx, q


def _pages(tokens, page):
    return -(-tokens // page)


# --------------------------------------------------------------------------
# inputs


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s = dict(case)

    if case["op"] == "plan":
        ctx, q = _lens(case)
        page = case["page"]
        width = max(_pages(c + n, page) for c, n in zip(ctx, q)) + 2
        held = sum(_pages(c, page) for c in ctx)
        need = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(ctx, q))
        perm = torch.randperm(held + need + 64, generator=g, device=dev).to(torch.int32)
        # the requests' own pages stand in their rows, unused entries are -1
        owned = torch.arange(width, device=dev)[None, :] < ints([_pages(c, page) for c in ctx])[:, None]
        table = torch.full((case["batch"], width), -1, dtype=torch.int32, device=dev)
        table[owned] = perm[:held]
        s.update(context_lens=ints(ctx), query_lens=ints(q), block_tables=table, free_pages=perm[held:].contiguous(),
                 num_tokens=sum(q))
        return s

    if case["op"] == "rope":
        t, hq, hk, d, page = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "page"))
        dt = DTYPES[case["dtype"]]
        # one row of the fused projection holds q | k | v
        qkv = randn(t, (hq + 2 * hk) * d).to(dt)
        n_pos = 16384
        freq = 500000.0 ** (-torch.arange(0, case["rot"], 2, device=dev, dtype=torch.float64) / case["rot"])
        angle = torch.arange(n_pos, device=dev, dtype=torch.float64)[:, None] * freq
        first = int(torch.randint(0, n_pos - t + 1, (1,), generator=g, device=dev))
        pages = _pages(t, page) + 3
        at = torch.arange(t, device=dev)
        order = torch.randperm(pages, generator=g, device=dev)
        s.update(qkv=qkv, cos=angle.cos().float(), sin=angle.sin().float(),
                 positions=(first + at).to(torch.int32), slots=order[at // page] * page + at % page,
                 k_cache=randn(pages, page, hk, d).to(dt), v_cache=randn(pages, page, hk, d).to(dt))
        return s

    if case["op"] == "attn":
        ctx, q = _lens(case)
        hq, hk, d, page = (case[k] for k in ("heads", "kv_heads", "dim", "page"))
        dt = DTYPES[case["dtype"]]
        total = [c + n for c, n in zip(ctx, q)]
        counts = [_pages(n, page) for n in total]
        pages = sum(counts) + 2
        width = max(max(counts), 1)
        table = torch.zeros(case["batch"], width, dtype=torch.int32, device=dev)
        owned = torch.arange(width, device=dev)[None, :] < ints(counts)[:, None]
        table[owned] = torch.randperm(pages, generator=g, device=dev)[:sum(counts)].to(torch.int32)
        cu = [0]
        for n in q:
            cu.append(cu[-1] + n)
        # scores with a spread of 2: some keys of a row matter much more than the rest
        s.update(q=(2.0 * randn(cu[-1], hq, d)).to(dt), k_cache=randn(pages, page, hk, d).to(dt),
                 v_cache=randn(pages, page, hk, d).to(dt), block_tables=table, seq_lens=ints(total),
                 cu_seqlens=ints(cu), max_query_len=max(q), scale_qk=d ** -0.5)
        return s

    t, e = case["tokens"], case["experts"]
    s.update(logits=randn(t, e).to(DTYPES[case["dtype"]]),
             balance=0.1 * randn(e) if case["bias"] else None)
    return s


# --------------------------------------------------------------------------
# one pass


def run(s):
    if own:
        return _run_own(s)
    return {"plan": _plan, "rope": _rope, "attn": _attn, "route": _route}[s["op"]](s)


def _run_own(s):
    from gmlx_b200 import kq
    if s["op"] == "plan":
        p = kq.paged_plan(s["context_lens"], s["query_lens"], s["block_tables"], s["free_pages"], s["page"],
                          s["num_tokens"])
        return {"block_tables": s["block_tables"], "cu_seqlens": p.cu_seqlens, "seq_lens": p.seq_lens,
                "slots": p.slots, "positions": p.positions, "pages_used": p.pages_used}
    if s["op"] == "rope":
        q, k, v = _split(s)
        rotated = kq.rope_kv_write(q, k, v, s["cos"], s["sin"], s["positions"], s["k_cache"], s["v_cache"], s["slots"],
                                   interleaved=s["interleaved"])
        return {"q": rotated, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if s["op"] == "attn":
        out = kq.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_tables"], s["seq_lens"], s["cu_seqlens"],
                                 s["max_query_len"], scale=s["scale_qk"], window=s["window"], softcap=s["softcap"],
                                 return_lse=s["lse"])
        return {"out": out[0], "lse": out[1]} if s["lse"] else {"out": out}
    idx, weights = kq.moe_route(s["logits"], s["k"], scoring=s["scoring"], bias=s["balance"], n_groups=s["groups"],
                                topk_groups=s["top_groups"], norm_topk_prob=s["norm"], scale=s["scale"])
    return {"experts": idx, "weights": weights}


def _plan(s):
    """Request b holds ceil(ctx/page) pages and needs ceil((ctx+new)/page); the
    missing ones come from the free list in request order.  Token i of request
    b stands at position ctx + i, in slot page_id * page + position % page."""
    page, table, free = s["page"], s["block_tables"], s["free_pages"]
    ctx, new = s["context_lens"].long(), s["query_lens"].long()
    ends = new.cumsum(0)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends])
    total = ctx + new
    held, wanted = (ctx + page - 1) // page, (total + page - 1) // page
    need = wanted - held
    first = need.cumsum(0) - need
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    taken = (col >= held[:, None]) & (col < wanted[:, None])
    src = (first[:, None] + col - held[:, None]).clamp(0, free.shape[0] - 1)
    table.copy_(torch.where(taken, free[src], table))
    t = torch.arange(s["num_tokens"], device=table.device)
    req = torch.searchsorted(ends, t, right=True)
    pos = ctx[req] + t - cu[req]
    slots = table[req, pos // page].long() * page + pos % page
    return {"block_tables": table, "cu_seqlens": cu.int(), "seq_lens": total.int(), "slots": slots,
            "positions": pos.int(), "pages_used": need.sum().int().reshape(1)}


def _split(s):
    hq, hk, d = s["heads"], s["kv_heads"], s["dim"]
    qkv = s["qkv"].view(s["tokens"], hq + 2 * hk, d)
    return qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]


def _rotate(x, cos, sin, rot, interleaved):
    """The first `rot` values of each head turn by the token's angles, in pairs
    (2i, 2i+1) where interleaved, else (i, i + rot/2); the rest stay."""
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _rope(s):
    q, k, v = _split(s)
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None, :], s["sin"][at][:, None, :]
    kc, vc = s["k_cache"], s["v_cache"]
    kc.view(-1, s["kv_heads"], s["dim"])[s["slots"]] = _rotate(k.float(), cos, sin, s["rot"], s["interleaved"]).to(kc.dtype)
    vc.view(-1, s["kv_heads"], s["dim"])[s["slots"]] = v
    return {"q": _rotate(q.float(), cos, sin, s["rot"], s["interleaved"]).to(q.dtype), "k_cache": kc, "v_cache": vc}


def _attn(s):
    """Row i of a request with n new tokens and L in all sees the keys
    [limit - window, limit) with limit = L - n + i + 1 (no lower bound where
    window is 0).  The batch is padded to its longest request."""
    q, table, seq, cu = s["q"], s["block_tables"].long(), s["seq_lens"].long(), s["cu_seqlens"].long()
    tokens, hq, d = q.shape
    hk, dev = s["kv_heads"], q.device
    b = table.shape[0]
    n_new = cu[1:] - cu[:-1]
    row = torch.arange(s["max_query_len"], device=dev)
    src = (cu[:-1, None] + row).clamp(max=tokens - 1)
    qp = q[src].float().view(b, -1, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d) * s["scale_qk"]
    key = torch.arange(table.shape[1] * s["page"], device=dev)
    inside = (key < seq[:, None])[:, :, None, None]
    kp = torch.where(inside, s["k_cache"][table].flatten(1, 2).float(), 0.0).transpose(1, 2)
    vp = torch.where(inside, s["v_cache"][table].flatten(1, 2).float(), 0.0).transpose(1, 2)
    x = qp @ kp.transpose(-1, -2)
    if s["softcap"]:
        x = s["softcap"] * torch.tanh(x / s["softcap"])
    limit = (seq - n_new)[:, None] + row + 1
    seen = key < limit[..., None]
    if s["window"]:
        seen &= key >= limit[..., None] - s["window"]
    x = x.view(b, hk, hq // hk, -1, key.shape[0]).masked_fill_(~seen[:, None, None], -INF)
    top = x.amax(-1, keepdim=True)
    base = torch.where(top == -INF, 0.0, top)
    x.sub_(base).exp_()
    total = x.sum(-1, keepdim=True)
    y = (x.flatten(2, 3) @ vp).view(b, hk, hq // hk, -1, d) / torch.where(total == 0, 1.0, total)
    t = torch.arange(tokens, device=dev)
    req = torch.searchsorted(cu[1:], t, right=True)
    at = t - cu[req]
    out = y.permute(0, 3, 1, 2, 4)[req, at].reshape(tokens, hq, d).to(q.dtype)
    if not s["lse"]:
        return {"out": out}
    lse = (base + total.log()).squeeze(-1)
    return {"out": out, "lse": lse.permute(0, 3, 1, 2)[req, at].reshape(tokens, hq)}


def _route(s):
    """Scores p = softmax or sigmoid of the logits; the choice goes by p + bias
    (the sum of the two best of a group ranks the group), the weights are p of
    the chosen.  The softmax's sum is held in 64 bits, so that its 32-bit value,
    and with it each choice, does not hang on the order of the additions."""
    x = s["logits"].float()
    t, e = x.shape
    if s["scoring"] == "sigmoid":
        p = 1.0 / (1.0 + torch.exp(-x))
    else:
        ex = torch.exp(x - x.amax(-1, keepdim=True))
        p = ex / ex.double().sum(-1, keepdim=True).float()
    key = p if s["balance"] is None else p + s["balance"]
    if s["groups"] > 1:
        per = key.view(t, s["groups"], -1)
        two = per.sort(dim=-1, descending=True)[0][..., :2]
        rank = (two[..., 0] + two[..., 1]).sort(dim=-1, descending=True, stable=True)[1][:, :s["top_groups"]]
        kept = torch.zeros(t, s["groups"], dtype=torch.bool, device=x.device).scatter_(1, rank, True)
        key = per.masked_fill(~kept[..., None], -INF).view(t, e)
    idx = key.sort(dim=-1, descending=True, stable=True)[1][:, :s["k"]]
    w = p.gather(1, idx)
    if s["norm"]:
        w = w / w.sum(-1, keepdim=True)
    return {"experts": idx.int(), "weights": w * s["scale"]}


# --------------------------------------------------------------------------
# what a pass cannot do without


def _seen_pairs(n, length, window):
    """(query, key) pairs of a request with n new tokens of `length`."""
    if not window:
        return n * (length - n) + n * (n + 1) // 2
    short = max(0, min(n, window - (length - n)))  # rows whose window is not full yet
    first = length - n + 1
    return short * first + short * (short - 1) // 2 + (n - short) * window


def work(case):
    if case["op"] == "plan":
        ctx, q = _lens(case)
        page, t, b = case["page"], sum(q), case["batch"]
        new = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(ctx, q))
        old = sum(1 for c, n in zip(ctx, q) if n and c % page)  # the half-filled page that the first token joins
        return {"bytes": 8 * b + 4 * old + 8 * new + 12 * t + 4 * (b + 1) + 4 * b + 4, "flops": 0}
    if case["op"] == "rope":
        t, hq, hk, d, rot = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "rot"))
        return {"bytes": t * (2 * (hq + 2 * hk) * d * 2 + 4 * rot + 12), "flops": t * (hq + hk) * rot * 3}
    if case["op"] == "attn":
        ctx, q = _lens(case)
        hq, hk, d, w = (case[k] for k in ("heads", "kv_heads", "dim", "window"))
        keys = sum(0 if not n else min(c + n, w + n - 1) if w else c + n for c, n in zip(ctx, q))
        pairs = sum(_seen_pairs(n, c + n, w) for c, n in zip(ctx, q))
        data = 2 * sum(q) * hq * d * 2 + 2 * keys * hk * d * 2 + 4 * (keys // case["page"] + 2 * len(q) + 1)
        return {"bytes": data + (4 * sum(q) * hq if case["lse"] else 0), "flops": 4 * pairs * hq * d}
    t, e, k = case["tokens"], case["experts"], case["k"]
    size = 4 if case["dtype"] == "f32" else 2
    return {"bytes": t * (e * size + 8 * k) + (4 * e if case["bias"] else 0), "flops": 4 * t * e}


# --------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "rope":
        t, hq, hk, d, rot = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "rot"))
        x = s["qkv"].double().view(t, hq + 2 * hk, d)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()][:, None, :]
        qk = x[:, :hq + hk].clone()
        even, odd = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
        z = torch.complex(qk[..., even], qk[..., odd]) * turn
        qk[..., even], qk[..., odd] = z.real, z.imag
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        page, off = s["slots"] // case["page"], s["slots"] % case["page"]
        kc[page, off], vc[page, off] = qk[:, hq:], x[:, hq + hk:]
        return {"q": qk[:, :hq].contiguous(), "k_cache": kc, "v_cache": vc}
    if case["op"] == "attn":
        return _exact_attn(case, s)
    x = s["logits"].double()
    p = torch.softmax(x, -1) if case["scoring"] == "softmax" else torch.sigmoid(x)
    key = p + s["balance"].double() if case["bias"] else p.clone()
    t, e, g = case["tokens"], case["experts"], case["groups"]
    if g > 1:
        score = key.view(t, g, e // g).topk(2, -1).values.sum(-1)
        order = torch.argsort(-score, dim=-1, stable=True)
        out = torch.ones(t, g, dtype=torch.bool, device=x.device)
        out.scatter_(1, order[:, :case["top_groups"]], False)
        key[out.repeat_interleave(e // g, 1)] = -INF
    w = torch.gather(p, 1, torch.argsort(-key, dim=-1, stable=True)[:, :case["k"]])
    if case["norm"]:
        w = w / w.sum(-1, keepdim=True)
    return {"experts": None, "weights": w * case["scale"]}


def _exact_attn(case, s):
    ctx, new = _lens(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    cap, window, dev = case["softcap"], case["window"], s["q"].device
    out = torch.zeros(sum(new), hq, d, dtype=torch.float64, device=dev)
    lse = torch.full((sum(new), hq), -INF, dtype=torch.float64, device=dev)
    start = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        if n == 0:
            continue
        length = c + n
        pages = s["block_tables"][r, :_pages(length, case["page"])].long()
        limit = torch.arange(c + 1, length + 1, device=dev)[:, None]
        key = torch.arange(length, device=dev)[None, :]
        hidden = (key >= limit) | (key < limit - window) if window else key >= limit
        for j in range(hk):
            k = s["k_cache"][pages, :, j].reshape(-1, d)[:length].double()
            v = s["v_cache"][pages, :, j].reshape(-1, d)[:length].double()
            for h in range(j * (hq // hk), (j + 1) * (hq // hk)):
                x = s["q"][start:start + n, h].double() @ k.t() * s["scale_qk"]
                if cap:
                    x = cap * torch.tanh(x / cap)
                x.masked_fill_(hidden, -INF)
                lse[start:start + n, h] = torch.logsumexp(x, -1)
                out[start:start + n, h] = torch.softmax(x, -1) @ v
        start += n
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
