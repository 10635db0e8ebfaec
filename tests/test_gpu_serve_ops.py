"""The serving-step operators against plain implementations in 64 bits.

Tolerances, from the formats (u = 2^-8 for bf16, 2^-11 for fp16: half a unit in
the last place, relative, of 8 and 11 bits):

* rotary embedding: f32 arithmetic and one rounding, so u * |x| plus the f32
  error of two products (2^-22 of |a| + |b|), of which cancellation leaves all.
* attention: one rounding of each probability and one of the result, each at
  most u of sum_j p_j |v_j|; the scores' f32 dot products err by at most
  d = (D + 8) 2^-24 * scale * max_j sum_i |q_i k_ji|, which moves each p by a
  factor within 1 +- 2d; 2^-18 for exponentials and sums.  fp16 probabilities
  below its normal range err by 2^-25 each instead.
* lse: d + 2^-18 (1 + |lse|).
* routing weights: 8 f32 roundings, 2^-20 relative; indices exactly.
"""
import math

import pytest
import torch

from gmlx_b200 import _lib, kq

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, FP = torch.bfloat16, torch.float16
INF = float("inf")


def slow(fn, *a, **k):
    """The call without the native fast path."""
    saved = kq._EXT
    kq._EXT = False
    try:
        return fn(*a, **k)
    finally:
        kq._EXT = saved


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# --------------------------------------------------------------------------
# plan


def plan_ref(ctx, new, table, free, page, tokens):
    table = [list(r) for r in table]
    cu, slots, pos, used = [0], [], [], 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        held, want = -(-c // page), -(-(c + n) // page)
        for col in range(held, want):
            if col < len(table[b]):
                table[b][col] = free[used] if used < len(free) else -1
            used += 1
        for p in range(c, c + n):
            col = p // page
            pid = table[b][col] if col < len(table[b]) else -1
            slots.append(pid * page + p % page if pid >= 0 else -1)
            pos.append(p)
        cu.append(cu[-1] + n)
    pad = tokens - len(slots)
    return table, cu, [c + n for c, n in zip(ctx, new)], slots + [-1] * pad, pos + [0] * pad, used


@pytest.mark.parametrize("batch,q_max,ctx_max,page,pad", [
    (1, 1, 0, 16, 0), (1, 700, 33, 16, 5), (3, 5, 7, 1, 0), (64, 1, 500, 16, 0), (1023, 3, 40, 7, 2),
    (1025, 9, 100, 24, 0), (5000, 2, 9, 4, 11), (8192, 1, 3, 2, 0), (7, 300, 1000, 128, 64)])
def test_plan(cuda, batch, q_max, ctx_max, page, pad):
    g = torch.Generator().manual_seed(batch * 7 + page)
    ctx = torch.randint(0, ctx_max + 1, (batch,), generator=g).tolist()
    new = torch.randint(0, q_max + 1, (batch,), generator=g).tolist()
    width = max(-(-(c + n) // page) for c, n in zip(ctx, new)) + 1
    ids = torch.randperm(batch * width + 3, generator=g).tolist()
    table, at = [], 0
    for c in ctx:
        held = -(-c // page)
        table.append(ids[at:at + held] + [-7] * (width - held))
        at += held
    free, tokens = ids[at:], sum(new) + pad
    ref = plan_ref(ctx, new, table, free, page, tokens)
    for call in (kq.paged_plan, lambda *a: slow(kq.paged_plan, *a)):
        wide = i32([r + [99, 99] for r in table], cuda)  # the table as a view of a wider one
        t = wide[:, :width]
        p = call(i32(ctx, cuda), i32(new, cuda), t, i32(free, cuda), page, tokens)
        assert t.tolist() == ref[0] and (wide[:, width:] == 99).all()
        assert p.cu_seqlens.tolist() == ref[1] and p.seq_lens.tolist() == ref[2]
        assert p.slots.tolist() == ref[3] and p.positions.tolist() == ref[4]
        assert p.pages_used.tolist() == [ref[5]]
        assert p.slots.dtype == torch.int64 and p.positions.dtype == torch.int32
    assert kq.workspace_error() == 0


def test_plan_empty_batch(cuda):
    e = torch.empty(0, dtype=torch.int32, device=cuda)
    p = kq.paged_plan(e, e, e.view(0, 0), e, 16, 3)
    assert p.cu_seqlens.tolist() == [0] and p.slots.tolist() == [-1] * 3 and p.pages_used.tolist() == [0]
    assert kq.workspace_error() == 0


def test_plan_out_of_pages_and_of_table(cuda):
    ctx, new, table, free = [3, 0], [4, 6], [[5, -1, -1], [-1, -1, -1]], [8, 9]
    t = i32(table, cuda)
    p = kq.paged_plan(i32(ctx, cuda), i32(new, cuda), t, i32(free, cuda), 4, 10)
    ref = plan_ref(ctx, new, table, free, 4, 10)  # the second request's second page is missing
    assert t.tolist() == ref[0] == [[5, 8, -1], [9, -1, -1]]
    assert p.slots.tolist() == ref[3] and p.slots.tolist()[-2:] == [-1, -1] and p.pages_used.tolist() == [3]
    assert kq.workspace_error() == 21
    t = i32([[5]], cuda)  # no room in the row
    p = kq.paged_plan(i32([3], cuda), i32([4], cuda), t, i32([1, 2], cuda), 4, 4)
    assert t.tolist() == [[5]] and p.slots.tolist() == [23, -1, -1, -1]
    assert kq.workspace_error() == 21 and kq.workspace_error() == 0


@pytest.mark.parametrize("ctx,new,tokens", [([-1, 2], [1, 1], 2), ([0, 0], [2, -3], 2), ([0, 0], [3, 3], 5),
                                            ([2 ** 31 - 1, 0], [1, 1], 2), ([0] * 2048, [2 ** 30] * 2048, 4)])
def test_plan_contradictory_lengths_are_reported(cuda, ctx, new, tokens):
    t = torch.full((len(ctx), 4), -1, dtype=torch.int32, device=cuda)
    kq.paged_plan(i32(ctx, cuda), i32(new, cuda), t, i32(list(range(16)), cuda), 4, tokens)
    assert kq.workspace_error() == 20 and kq.workspace_error() == 0


def test_plan_refusals(cuda):
    a, t, f = i32([1, 2], cuda), i32([[0, 1], [2, 3]], cuda), i32([4], cuda)
    for bad in ((a.long(), a, t, f, 4, 2), (a, a[:1], t, f, 4, 2), (a, a, t[:1], f, 4, 2), (a, a, t.long(), f, 4, 2),
                (a, a, t, f, 0, 2), (a, a, t, f, 4, -1), (a, a, t.t(), f, 4, 2), (a.cpu(), a, t, f, 4, 2),
                (a, a, t, f.view(1, 1), 4, 2)):
        with pytest.raises(ValueError):
            kq.paged_plan(*bad)
    big = torch.zeros(8193, dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="8192"):
        kq.paged_plan(big, big, big.view(-1, 1), f, 4, 2)


# --------------------------------------------------------------------------
# rotary embedding and cache write


def rope_ref(x, cos, sin, rot, inter):
    x = x.double().clone()
    e, o = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., e].clone(), x[..., o].clone()
    c, s = cos.double()[:, None], sin.double()[:, None]
    x[..., e], x[..., o] = a * c - b * s, b * c + a * s
    size = torch.zeros_like(x)
    size[..., e] = size[..., o] = a.abs() + b.abs()
    return x, size


@pytest.mark.parametrize("t,hq,hk,d,rot,page,dtype,inter,layout", [
    (1, 32, 8, 128, 128, 16, BF, False, "fused"), (1, 1, 1, 16, 16, 1, FP, True, "plain"),
    (77, 32, 8, 128, 128, 16, BF, True, "fused"), (600, 6, 2, 64, 32, 24, FP, False, "fused"),
    (33, 5, 1, 256, 256, 64, BF, False, "heads_first"), (9, 3, 3, 80, 48, 5, BF, True, "plain"),
    (130, 7, 7, 96, 0, 32, FP, False, "plain"), (3, 2, 1, 1024, 1024, 2, BF, False, "plain"),
    (1200, 40, 8, 64, 64, 16, FP, False, "fused")])
def test_rope_kv_write(cuda, t, hq, hk, d, rot, page, dtype, inter, layout):
    torch.manual_seed(t + d)
    if layout == "fused":
        qkv = torch.randn(t, hq + 2 * hk, d, device=cuda).to(dtype)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    elif layout == "heads_first":
        q, k, v = (torch.randn(h, t, d, device=cuda).to(dtype).transpose(0, 1) for h in (hq, hk, hk))
    else:
        q, k, v = (torch.randn(t, h, d, device=cuda).to(dtype) for h in (hq, hk, hk))
    n_pos = 500
    angle = 10 * torch.randn(n_pos, rot // 2, device=cuda)
    cos, sin = angle.cos(), angle.sin()
    pos = torch.randint(0, n_pos, (t,), device=cuda, dtype=torch.int32)
    pages = t // page + 3
    slots = torch.randperm(pages * page, device=cuda)[:t]
    slots[::5] = -1  # padding tokens are turned but not stored
    shape = (pages, page, hk, d)
    kc, vc = torch.randn(2, *shape, device=cuda).to(dtype)
    if layout == "heads_first":  # pages hold their heads first
        kc, vc = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc))
    k0, v0 = kc.clone(), vc.clone()
    out = kq.rope_kv_write(q, k, v, cos, sin, pos, kc, vc, slots, interleaved=inter)
    p = pos.long()
    for got, x in ((out, q), (None, k)):
        ref, size = rope_ref(x, cos[p], sin[p], rot, inter)
        tol = U[dtype] * ref.abs() + 2.0 ** -22 * size + (2.0 ** -25 if dtype == FP else 0)
        if got is not None:
            assert got.shape == (t, hq, d) and got.is_contiguous()
            assert ((got.double() - ref).abs() <= tol).all()
        else:
            kept = slots >= 0
            pg, off = slots[kept] // page, slots[kept] % page
            assert ((kc[pg, off].double() - ref[kept]).abs() <= tol[kept]).all()
            assert torch.equal(vc[pg, off], v[kept])
            rest = torch.ones(pages, page, dtype=torch.bool, device=cuda)
            rest[pg, off] = False
            assert torch.equal(kc[rest], k0[rest]) and torch.equal(vc[rest], v0[rest])
    kc2, vc2 = k0.clone(), v0.clone()
    out2 = slow(kq.rope_kv_write, q, k, v, cos, sin, pos, kc2, vc2, slots, interleaved=inter)
    assert torch.equal(out, out2) and torch.equal(kc, kc2) and torch.equal(vc, vc2)
    assert kq.workspace_error() == 0


def test_rope_reports_positions_and_slots_outside(cuda):
    q, k, v = (torch.randn(2, h, 64, device=cuda).to(BF) for h in (4, 2, 2))
    cos = torch.ones(10, 32, device=cuda)
    kc, vc = torch.zeros(2, 2, 4, 2, 64, device=cuda, dtype=BF)
    args = lambda p, s: (q, k, v, cos, cos * 0, i32(p, cuda), kc, vc, torch.tensor(s, device=cuda))  # noqa: E731
    kq.rope_kv_write(*args([0, 10], [0, 1]))
    assert kq.workspace_error() == 22
    kq.rope_kv_write(*args([0, -1], [0, 1]))
    assert kq.workspace_error() == 22
    kc.zero_()
    kq.rope_kv_write(*args([0, 1], [8, 3]))
    assert kq.workspace_error() == 22 and kq.workspace_error() == 0
    assert torch.equal(kc[0, 3], k[1]) and kc.count_nonzero() == k[1].count_nonzero()


def test_rope_refusals(cuda):
    q, k, v = (torch.randn(2, h, 64, device=cuda).to(BF) for h in (4, 2, 2))
    cos, pos, slot = torch.ones(10, 32, device=cuda), i32([0, 1], cuda), torch.tensor([0, 1], device=cuda)
    kc, vc = torch.zeros(2, 2, 4, 2, 64, device=cuda, dtype=BF)
    good = dict(q=q, k=k, v=v, cos=cos, sin=cos, positions=pos, k_cache=kc, v_cache=vc, slots=slot)
    kq.rope_kv_write(**good)
    for name, bad in (("q", q.half()), ("k", k[:1]), ("v", v[:, :1]), ("cos", cos.half()), ("sin", cos[:, :16]),
                      ("positions", pos.long()), ("slots", slot.int()), ("v_cache", vc.half()), ("k_cache", kc.float()),
                      ("v_cache", vc.transpose(1, 2).contiguous().transpose(1, 2)), ("q", q.cpu()), ("k_cache", kc[0])):
        with pytest.raises(ValueError):
            kq.rope_kv_write(**{**good, name: bad})
    for rot in (8, 40):  # 2 * rot / 2 values: not a multiple of 16, more than the head
        with pytest.raises(ValueError):
            kq.rope_kv_write(**{**good, "cos": torch.ones(10, rot, device=cuda)[:, :rot if rot > 8 else 4],
                                "sin": torch.ones(10, rot, device=cuda)[:, :rot if rot > 8 else 4]})


# --------------------------------------------------------------------------
# attention


def attn_inputs(dev, lens, hq, hk, d, page, dtype, seed=0, pad=0, layout="rows", extra_width=0):
    """lens: (new, total) of each request.  Whatever the cache holds outside the
    requests is NaN, and unused table entries point far outside it."""
    g = torch.Generator(device=dev).manual_seed(seed)
    counts = [-(-n // page) for _, n in lens]
    pages = sum(counts) + 3
    width = max(counts + [1]) + extra_width
    order = torch.randperm(pages, generator=g, device=dev).tolist()
    table = torch.full((len(lens), width), 2 ** 30, dtype=torch.int32, device=dev)
    kv = torch.full((2, pages, page, hk, d), float("nan"), dtype=dtype, device=dev)
    at = 0
    for b, (_, total) in enumerate(lens):
        ids = order[at:at + counts[b]]
        at += counts[b]
        if ids:
            table[b, :len(ids)] = i32(ids, dev)
            rows = torch.randn(2, total, hk, d, generator=g, device=dev).to(dtype)
            for j, pid in enumerate(ids):
                r = rows[:, j * page:(j + 1) * page]
                kv[:, pid, :r.shape[1]] = r
    cu = [0]
    for n, _ in lens:
        cu.append(cu[-1] + n)
    q = (2 * torch.randn(cu[-1] + pad, hq, d, generator=g, device=dev)).to(dtype)
    kc, vc = kv[0], kv[1]
    if layout == "heads":
        kc, vc = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc))
    elif layout == "interleaved":  # one tensor [pages, page, 2, heads, dim]
        both = torch.stack([kc, vc], 2)
        kc, vc = both[:, :, 0], both[:, :, 1]
    return q, kc, vc, table, i32([n for _, n in lens], dev), i32(cu, dev)


def attn_ref(q, kc, vc, table, seq, cu, scale, window, softcap, causal):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits."""
    t, hq, d = q.shape
    hk, page = kc.shape[2], kc.shape[1]
    u = U[q.dtype]
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((t, hq), -INF, dtype=torch.float64, device=q.device)
    tol, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    cu, seq = cu.tolist(), seq.tolist()
    for b, total in enumerate(seq):
        n = cu[b + 1] - cu[b]
        if n == 0 or total == 0:
            continue
        ids = table[b, :-(-total // page)].long()
        key = torch.arange(total, device=q.device)[None]
        limit = (torch.arange(n, device=q.device) + total - n + 1)[:, None] if causal else torch.full((n, 1), total, device=q.device)
        seen = key < limit
        if window:
            seen &= key >= limit - window
        live = seen.any(1)
        for h in range(hq):
            k = kc[ids][:, :, h // (hq // hk)].reshape(-1, d)[:total].double()
            v = vc[ids][:, :, h // (hq // hk)].reshape(-1, d)[:total].double()
            x = q[cu[b]:cu[b + 1], h].double()
            s = x @ k.t() * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            s = s.masked_fill(~seen, -INF)
            p = torch.where(live[:, None], torch.softmax(s, -1), 0.0).nan_to_num(0.0)
            rows = slice(cu[b], cu[b + 1])
            out[rows, h] = p @ v
            lse[rows, h] = torch.logsumexp(s, -1)
            dd = (d + 8) * 2.0 ** -24 * scale * (x.abs() @ k.abs().t()).masked_fill(~seen, 0).amax(-1, keepdim=True)
            tol[rows, h] = (2 * u + 2 * dd + 2.0 ** -18) * (p @ v.abs())
            if q.dtype == FP:  # probabilities under the normal range, relative to the largest; results too
                tol[rows, h] += seen.sum(-1, keepdim=True) * 2.0 ** -25 * p.amax(-1, keepdim=True) * v.abs().max() + 2.0 ** -25
            tol_l[rows, h] = torch.where(live, dd[:, 0] + 2.0 ** -18 * (1 + lse[rows, h].abs()), 0.0)
    return out, lse, tol, tol_l


def check_attn(args, max_q, scale=None, window=0, softcap=0.0, causal=True):
    q = args[0]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    ref, ref_l, tol, tol_l = attn_ref(*args, scale, window, softcap, causal)
    out, lse = kq.paged_attention(*args, max_q, scale=scale, window=window, softcap=softcap, causal=causal, return_lse=True)
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    off = (out.double() - ref).abs()
    assert (off <= tol).all(), (off - tol).max().item()
    none = ref_l == -INF
    assert (lse[none] == -INF).all() and (out[none] == 0).all()
    off = (lse.double() - ref_l).abs()[~none]
    assert (off <= tol_l[~none]).all(), (off - tol_l[~none]).max().item()
    assert kq.workspace_error() == 0
    return out, lse


DECODE = [
    # lens, hq, hk, d, page, dtype, window, softcap
    ([(1, 1)], 1, 1, 64, 1, BF, 0, 0.0),
    ([(1, 17)], 4, 4, 128, 16, FP, 0, 0.0),
    ([(1, 999)], 32, 8, 128, 16, BF, 0, 0.0),
    ([(1, 64), (1, 65), (1, 63), (1, 1), (1, 300)], 8, 2, 128, 16, BF, 0, 0.0),
    ([(1, 5000), (1, 3)], 16, 1, 64, 32, FP, 0, 0.0),
    ([(2, 700), (4, 4), (3, 1000)], 8, 2, 128, 24, BF, 0, 30.0),
    ([(1, 200)] * 40, 7, 1, 256, 7, BF, 50, 0.0),
    ([(1, 3000), (1, 17), (1, 128)], 10, 2, 128, 128, FP, 129, 20.0),
    ([(4, 20000)], 4, 1, 128, 64, BF, 0, 0.0),
    ([(1, 130)] * 3, 96, 2, 64, 8, BF, 0, 0.0),  # 48 query heads a kv head
]


@pytest.mark.parametrize("lens,hq,hk,d,page,dtype,window,softcap", DECODE)
def test_attention_few_tokens(cuda, lens, hq, hk, d, page, dtype, window, softcap):
    check_attn(attn_inputs(cuda, lens, hq, hk, d, page, dtype), max(n for n, _ in lens), window=window, softcap=softcap)


CHUNK = [
    ([(17, 17)], 4, 1, 128, 16, BF, 0, 0.0),
    ([(64, 64)], 8, 8, 64, 16, FP, 0, 0.0),
    ([(129, 129)], 4, 2, 128, 16, BF, 0, 0.0),
    ([(300, 1000)], 8, 2, 128, 32, BF, 0, 0.0),
    ([(512, 512)], 6, 2, 128, 64, FP, 0, 0.0),
    ([(33, 5000)], 8, 1, 128, 16, BF, 0, 0.0),
    ([(200, 900), (1, 700), (0, 40), (37, 37), (1, 1), (90, 2000)], 10, 2, 64, 24, FP, 100, 50.0),
    ([(250, 777), (60, 60)], 7, 1, 256, 8, BF, 0, 0.0),
    ([(100, 300), (150, 150)], 14, 2, 128, 1, BF, 0, 0.0),
    ([(700, 1500)], 3, 3, 128, 100, BF, 333, 0.0),
    ([(40, 400)] * 9, 20, 4, 128, 128, FP, 0, 0.0),
    ([(65, 4000), (2, 3000)], 64, 2, 64, 16, BF, 0, 0.0),
    ([(260, 260)], 2, 1, 128, 256, BF, 7, 0.0),
]


@pytest.mark.parametrize("lens,hq,hk,d,page,dtype,window,softcap", CHUNK)
def test_attention_chunk(cuda, lens, hq, hk, d, page, dtype, window, softcap):
    check_attn(attn_inputs(cuda, lens, hq, hk, d, page, dtype), max(n for n, _ in lens), window=window, softcap=softcap)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(1, 300), (1, 31)], [(150, 300), (1, 77), (40, 40)]])
def test_attention_not_causal(cuda, lens, d):
    check_attn(attn_inputs(cuda, lens, 8, 2, d, 16, BF), max(n for n, _ in lens), causal=False)


@pytest.mark.parametrize("layout", ["heads", "interleaved"])
@pytest.mark.parametrize("lens", [[(1, 300), (3, 31)], [(150, 300), (1, 77), (40, 40)]])
def test_attention_cache_layouts_and_strided_queries(cuda, lens, layout):
    args = attn_inputs(cuda, lens, 8, 2, 128, 16, BF, layout=layout, extra_width=3)
    out, lse = check_attn(args, max(n for n, _ in lens))
    q = args[0]
    wide = torch.zeros(q.shape[0], 12, 128, dtype=BF, device=cuda)  # q | k | v of a fused projection
    wide[:, :8] = q
    first = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(q.numel() + 1, dtype=BF, device=cuda)[1:].view(q.shape).copy_(q)  # not 16-byte aligned
    table = torch.cat([args[3], args[3]], 1)[:, :args[3].shape[1]]
    for other in (wide[:, :8], first, odd):
        again = kq.paged_attention(other, *args[1:3], table, *args[4:], max(n for n, _ in lens), return_lse=True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    again = slow(kq.paged_attention, *args, max(n for n, _ in lens), return_lse=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(3, 2), (1, 0), (2, 2)], [(200, 50), (40, 0), (0, 9), (130, 129)]])
def test_attention_rows_without_keys_and_padding(cuda, lens, d):
    """More new tokens than keys: the first rows see none.  Tokens behind the
    last request are padding."""
    args = attn_inputs(cuda, lens, 4, 2, d, 16, BF, pad=5)
    out, lse = check_attn(args, max(n for n, _ in lens))
    assert (out[-5:] == 0).all() and (lse[-5:] == -INF).all()


def test_attention_no_requests(cuda):
    q = torch.randn(3, 4, 64, device=cuda).to(BF)
    kc = torch.zeros(1, 16, 2, 64, device=cuda, dtype=BF)
    e = torch.empty(0, dtype=torch.int32, device=cuda)
    out = kq.paged_attention(q, kc, kc, e.view(0, 0), e, i32([0], cuda), 1)
    assert (out == 0).all()
    assert kq.paged_attention(q[:0], kc, kc, e.view(0, 0), e, i32([0], cuda), 1).shape == (0, 4, 64)
    assert kq.workspace_error() == 0


@pytest.mark.parametrize("max_q", [0, 1, 10 ** 6])
def test_attention_hint_only_picks_kernels(cuda, max_q):
    check_attn(attn_inputs(cuda, [(150, 600), (1, 50), (5, 90)], 8, 2, 128, 16, BF), max_q)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens", [[(1, 2000)], [(130, 2000)]])
def test_attention_large_scores(cuda, lens, dtype):
    """Scores of a few hundred: one key takes the row, and nothing overflows."""
    args = attn_inputs(cuda, lens, 4, 2, 128, 16, dtype, seed=5)
    check_attn((args[0] * 8,) + args[1:], lens[0][0], scale=1.0)


@pytest.mark.parametrize("lens", [[(1, 1500)], [(140, 1500)]])
def test_attention_growing_maximum(cuda, lens):
    """Scores that grow along the keys make every tile raise the running maximum;
    falling ones never do."""
    for sign in (1.0, -1.0):
        q, kc, vc, table, seq, cu = attn_inputs(cuda, lens, 4, 1, 128, 16, BF, seed=3)
        pos = torch.arange(1504, device=cuda).view(94, 16)
        kc.nan_to_num_(0.0)
        kc[table[0].long(), :, 0, 0] = (sign * 0.05 * pos).to(BF)
        q[..., 0] = 4.0
        check_attn((q, kc, vc, table, seq, cu), lens[0][0])


@pytest.mark.parametrize("d,dtype", [(64, FP), (64, BF), (128, FP), (128, BF), (256, BF)])
@pytest.mark.parametrize("lens,window", [([(700, 700)], 0), ([(1, 40)] * 3 + [(333, 900), (90, 90), (2, 2), (400, 401)], 170)])
def test_attention_more_pairs_than_blocks(cuda, lens, window, d, dtype):
    """Pairs of one key tile beside pairs of many, cut wherever an even run ends."""
    check_attn(attn_inputs(cuda, lens, 64, 8, d, 16, dtype), max(n for n, _ in lens), window=window)


@pytest.mark.parametrize("shift", [-40.0, 40.0])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attention_scores_far_from_zero(cuda, shift, dtype):
    """Every score of a row near `shift`: probabilities that leave the type's range unless
    they are taken relative to something near it."""
    args = attn_inputs(cuda, [(150, 520), (33, 33)], 4, 2, 64, 16, dtype)
    q, kc = args[0], args[1]
    q[..., 0], kc[..., 0] = 8.0, torch.where(kc[..., 0].isnan(), kc[..., 0], shift)  # adds 8 shift / 8
    check_attn(args, 150)


@pytest.mark.parametrize("lens", [[(1, 700), (2, 30)], [(130, 700), (2, 30)]])
def test_attention_reports_foreign_pages(cuda, lens):
    args = attn_inputs(cuda, lens, 4, 2, 128, 16, BF)
    good = kq.paged_attention(*args, 130)
    assert kq.workspace_error() == 0
    for page in (-1, 2 ** 30):
        table = args[3].clone()
        table[0, 7] = page
        got = kq.paged_attention(*args[:3], table, *args[4:], 130)
        assert kq.workspace_error() == 22 and kq.workspace_error() == 0
        assert torch.equal(got[lens[0][0]:], good[lens[0][0]:])  # the other request is untouched
        # the foreign page counts as zeros
        kz, vz = args[1].clone(), args[2].clone()
        kz[args[3][0, 7].long()] = 0
        vz[args[3][0, 7].long()] = 0
        assert torch.equal(got, kq.paged_attention(args[0], kz, vz, *args[3:], 130))


def test_attention_reports_contradictory_lengths(cuda):
    q, kc, vc, table, seq, cu = attn_inputs(cuda, [(4, 40), (3, 30)], 4, 2, 64, 16, BF)
    for s, c in (([40, 1000], [0, 4, 7]), ([40, -1], [0, 4, 7]), ([40, 30], [0, 4, 9]), ([40, 30], [0, 5, 4]),
                 ([40, 30], [-2, 4, 7])):
        kq.paged_attention(q, kc, vc, torch.zeros_like(table), i32(s, cuda), i32(c, cuda), 4)
        assert kq.workspace_error() == 20 and kq.workspace_error() == 0


def test_attention_offsets_past_32_bits(cuda):
    """The last pages of a cache of more than 2^32 values."""
    hk, d, page = 8, 128, 64
    pages = 2 ** 32 // (hk * d * page) + 40
    kc = torch.empty(pages, page, hk, d, dtype=BF, device=cuda)
    vc = torch.empty_like(kc)
    for lens in ([(1, 1000)], [(200, 1000)]):
        q, k0, v0, table, seq, cu = attn_inputs(cuda, lens, 16, hk, d, page, BF)
        kc[-k0.shape[0]:], vc[-k0.shape[0]:] = k0, v0
        a = kq.paged_attention(q, k0, v0, table, seq, cu, lens[0][0])
        b = kq.paged_attention(q, kc, vc, table + (pages - k0.shape[0]), seq, cu, lens[0][0])
        assert torch.equal(a, b)
    pos, slots = i32([0], cuda), torch.tensor([pages * page - 1], device=cuda)
    k, v = torch.randn(2, 1, hk, d, device=cuda).to(BF)
    one = torch.ones(1, d // 2, device=cuda)
    kq.rope_kv_write(k, k, v, one, one * 0, pos, kc, vc, slots)
    assert torch.equal(kc[-1, -1], k[0]) and torch.equal(vc[-1, -1], v[0])
    assert kq.workspace_error() == 0


def test_attention_repeats_bit_for_bit_on_any_stream(cuda):
    args = attn_inputs(cuda, [(1, 9000), (1, 100), (130, 3000)], 8, 2, 128, 16, BF)
    first = kq.paged_attention(*args, 130)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [kq.paged_attention(*args, 130) for _ in range(20)]
        err = kq.workspace_error()
    torch.cuda.current_stream().wait_stream(side)
    assert err == 0 and all(torch.equal(first, o) for o in outs)


def test_attention_in_a_graph_follows_its_lengths(cuda):
    """One captured call serves other lengths of the same buffers."""
    args = attn_inputs(cuda, [(1, 900), (1, 500)], 8, 2, 128, 16, BF)
    seq = args[4].clone()
    kq.paged_attention(*args[:4], seq, args[5], 1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        kq.paged_attention(*args[:4], seq, args[5], 1)  # the stream's workspace exists before the capture
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = kq.paged_attention(*args[:4], seq, args[5], 1)
    for lens in ([900, 500], [17, 400], [1, 0]):
        seq.copy_(i32(lens, cuda))
        g.replay()
        assert torch.equal(out, kq.paged_attention(*args[:4], i32(lens, cuda), args[5], 1))


def test_attention_refusals(cuda):
    q, kc, vc, table, seq, cu = attn_inputs(cuda, [(1, 40), (2, 30)], 4, 2, 64, 16, BF)
    good = dict(q=q, k_cache=kc, v_cache=vc, block_tables=table, seq_lens=seq, cu_seqlens=cu, max_query_len=2)
    kq.paged_attention(**good)
    for name, bad in (("q", q.float()), ("q", q.half()), ("q", q[..., :32]), ("q", q[:, :3]), ("q", q.cpu()),
                      ("k_cache", kc[0]), ("v_cache", vc.half()), ("v_cache", vc[:1]), ("block_tables", table.long()),
                      ("block_tables", table[:1]), ("seq_lens", seq.long()), ("seq_lens", seq[:1]),
                      ("cu_seqlens", cu[:2]), ("cu_seqlens", cu.long()), ("max_query_len", -1), ("window", -1),
                      ("softcap", -1.0), ("softcap", INF), ("scale", float("nan")), ("scale", INF)):
        with pytest.raises(ValueError):
            kq.paged_attention(**{**good, name: bad})
    with pytest.raises(ValueError, match="window"):
        kq.paged_attention(**good, window=5, causal=False)
    q96 = torch.zeros(3, 4, 96, dtype=BF, device=cuda)
    c96 = torch.zeros(4, 16, 2, 96, dtype=BF, device=cuda)
    with pytest.raises(ValueError, match="96"):
        kq.paged_attention(q96, c96, c96, table, seq, cu, 2)
    with pytest.raises(_lib.KQError):  # no workspace at the C entry: a status, not a fault
        c = kq._paged_cache("t", kc, vc)
        import ctypes
        _lib.check(_lib.load().kq_paged_attention(ctypes.byref(c), q.data_ptr(), 256, 64, 3, 4, table.data_ptr(), table.shape[1],
                                                  table.shape[1], seq.data_ptr(), cu.data_ptr(), 2, 2, 1.0, 1, 0, 0.0,
                                                  q.data_ptr(), None, None, 0, None))


# --------------------------------------------------------------------------
# routing


def route_ref(x, k, sigmoid, bias, groups, top, norm, scale):
    """Choice in f32, as defined (an exact function of the logits), weights in 64 bits."""
    t, e = x.shape
    x = torch.where(x.float().isnan(), -INF, x.float()).clamp(max=3.402823466e38)
    if sigmoid:
        p32 = 1.0 / (1.0 + torch.exp(-x))
        p = torch.sigmoid(x.double())
    else:
        top_x = x.amax(-1, keepdim=True)
        top_x = torch.where(top_x == -INF, 0.0, top_x)
        ex = torch.exp(x - top_x)
        s = ex.double().sum(-1, keepdim=True)
        p32 = torch.where(s > 0, ex / s.float(), 0.0)
        xd = (x.double() - top_x.double()).exp()
        p = torch.where(s > 0, xd / xd.sum(-1, keepdim=True), 0.0)
    key = p32 if bias is None else p32 + bias
    if groups > 1:
        per = key.view(t, groups, -1)
        two = per.sort(dim=-1, descending=True)[0][..., :2]
        order = (two[..., 0] + two[..., 1]).sort(dim=-1, descending=True, stable=True)[1][:, :top]
        kept = torch.zeros(t, groups, dtype=torch.bool, device=x.device).scatter_(1, order, True)
        key = per.masked_fill(~kept[..., None], -INF).view(t, e)
    idx = key.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    w = p.gather(1, idx)
    if norm:
        tot = w.sum(-1, keepdim=True)
        w = torch.where(tot > 0, w / tot, 0.0)
    return idx, w * scale


@pytest.mark.parametrize("t,e,k,sigmoid,bias,groups,top,norm,scale,dtype", [
    (1, 128, 8, False, False, 1, 1, True, 1.0, torch.float32), (1, 1, 1, False, False, 1, 1, True, 1.0, torch.float32),
    (64, 256, 8, True, True, 8, 4, True, 2.5, torch.float32), (4097, 256, 8, True, True, 8, 4, True, 2.5, BF),
    (130, 160, 6, False, True, 8, 3, False, 16.0, FP), (7, 100, 4, True, False, 1, 1, True, 1.0, BF),
    (33, 60, 4, False, False, 3, 2, True, 1.0, torch.float32), (5, 1024, 32, True, True, 32, 32, True, 1.0, FP),
    (19, 512, 10, False, True, 1, 1, True, 1.0, BF), (3, 8, 8, True, True, 4, 4, False, 1.0, BF),
    (1000, 64, 2, False, False, 1, 1, False, 1.0, BF), (12, 33, 3, True, True, 1, 1, True, 0.0, torch.float32)])
def test_route(cuda, t, e, k, sigmoid, bias, groups, top, norm, scale, dtype):
    torch.manual_seed(t + e)
    wide = torch.randn(t, e + 7, device=cuda).to(dtype)
    for x in (wide[:, :e], wide[:, :e].contiguous(), wide[:, 0:1].expand(t, e)):  # strided, dense, all equal
        b = 0.1 * torch.randn(e, device=cuda) if bias else None
        ref_i, ref_w = route_ref(x, k, sigmoid, b, groups, top, norm, scale)
        args = (x, k, "sigmoid" if sigmoid else "softmax", b, groups, top, norm, scale)
        idx, w = kq.moe_route(*args)
        assert idx.dtype == torch.int32 and w.dtype == torch.float32
        assert torch.equal(idx.long(), ref_i)
        assert ((w.double() - ref_w).abs() <= 2.0 ** -20 * ref_w.abs()).all()
        i2, w2 = slow(kq.moe_route, *args)
        assert torch.equal(idx, i2) and torch.equal(w, w2)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_masked_and_extreme_logits(cuda, sigmoid, groups):
    torch.manual_seed(1)
    x = torch.randn(8, 32, device=cuda)
    x[0, 3:] = -INF              # fewer open experts than k
    x[1] = -INF                  # none at all
    x[2, 5] = float("nan")       # counts as masked
    x[3, 7] = INF
    x[4] = torch.finfo(torch.float32).min
    x[5] *= 1e4
    x[6] = float("nan")
    for norm in (True, False):
        ref_i, ref_w = route_ref(x, 4, sigmoid, None, groups, groups, norm, 1.0)
        idx, w = kq.moe_route(x, 4, "sigmoid" if sigmoid else "softmax", None, groups, groups, norm)
        assert torch.equal(idx.long(), ref_i)
        assert torch.isfinite(w).all() and ((w.double() - ref_w).abs() <= 2.0 ** -20 * ref_w.abs() + 2.0 ** -120).all()
        assert (w[1] == 0).all() and (w[6] == 0).all()


def test_route_shapes_and_refusals(cuda):
    x = torch.randn(2, 3, 64, device=cuda)
    idx, w = kq.moe_route(x, 4)
    i2, w2 = kq.moe_route(x.view(6, 64), 4)
    assert idx.shape == w.shape == (2, 3, 4) and torch.equal(idx.view(6, 4), i2) and torch.equal(w.view(6, 4), w2)
    assert kq.moe_route(x[:0, 0], 4)[0].shape == (0, 4)
    b = torch.zeros(64, device=cuda)
    for kw in (dict(k=0), dict(k=33), dict(k=65), dict(k=4, scoring="relu"), dict(k=4, n_groups=5), dict(k=4, n_groups=64),
               dict(k=4, n_groups=4, topk_groups=5), dict(k=4, topk_groups=0), dict(k=20, n_groups=4, topk_groups=1),
               dict(k=4, bias=b[:32]), dict(k=4, bias=b.half()), dict(k=4, bias=b.cpu()), dict(k=4, scale=INF)):
        for shape in ((6, 64), (2, 3, 64)):
            with pytest.raises(ValueError):
                kq.moe_route(x.view(shape), **kw)
    with pytest.raises(ValueError):
        kq.moe_route(x.double(), 4)
    with pytest.raises(ValueError):
        kq.moe_route(torch.zeros(2, 1025, device=cuda), 4)
    with pytest.raises(ValueError, match="CUDA"):
        kq.moe_route(x.cpu(), 4)


def test_routed_experts_feed_the_expert_layer(cuda):
    """The router's outputs go straight into the quantized expert layer."""
    from gmlx_b200 import synth
    t, e, d, f, k = 5, 8, 512, 256, 2
    wg, wu = (torch.from_numpy(synth.random_weight("q4_k", e * f, d, seed=s).reshape(e, f, -1)).to(cuda) for s in (1, 2))
    wd = torch.from_numpy(synth.random_weight("q6_k", e * d, f, seed=3).reshape(e, d, -1)).to(cuda)
    torch.manual_seed(0)
    x = torch.randn(t, d, device=cuda).to(BF)
    idx, w = kq.moe_route(torch.randn(t, e, device=cuda), k, "sigmoid", 0.1 * torch.randn(e, device=cuda), 4, 2)
    y = kq.moe_expert_layer_local(x, idx, w, wg, wu, wd, "q4_k", "q6_k", out_dtype=torch.float32).double()
    ref = torch.zeros(t, d, dtype=torch.float64, device=cuda)
    g, u, o = (kq.dequantize(a, None, c).double() for a, c in ((wg, "q4_k"), (wu, "q4_k"), (wd, "q6_k")))
    for i in range(t):
        for j in range(k):
            n = int(idx[i, j])
            z = x[i].double()
            h = torch.nn.functional.silu(g[n] @ z) * (u[n] @ z)
            ref[i] += float(w[i, j]) * (o[n] @ h)
    assert (y - ref).abs().max() <= 1e-2 * ref.abs().max()
    assert math.isfinite(float(y.sum()))
