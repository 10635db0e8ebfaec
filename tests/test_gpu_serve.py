"""The serving step (``gmlx_b200.serve``) over several steps of mixed prompts and
single tokens: what each operator was given and gave is checked against plain
64-bit forms that know only the requests' history, with the operators' own
tolerances; what the layer does around them is repeated and must agree bit for bit."""
import pytest
import torch

from gmlx_b200 import kq, serve, synth

from test_gpu_serve_ops import BF, FP, U, attn_ref, rope_ref, route_ref

pytestmark = pytest.mark.gpu


def fill(module, seed):
    """Random wire bytes in every quantized weight, random norms and routers.  The
    bytes stand for weights far above trained ones, so the norms' gains are 2^-4:
    the experts' gate * up products then stay within fp16's range."""
    g = torch.Generator().manual_seed(seed)
    for i, m in enumerate(module.modules()):
        c = getattr(m, "kquant_type", None)
        if c is not None:
            rows = m.weight.numel() // m.weight.shape[-1]
            w = synth.random_weight(c, rows, m.in_dims, seed=seed * 100 + i)
            m.weight.copy_(torch.from_numpy(w).reshape(m.weight.shape))
    for name in ("attn_norm", "ffn_norm"):
        getattr(module, name).copy_(2.0 ** -4 * (1 + 0.1 * torch.randn(module.attn_norm.shape, generator=g)))
    module.gate.weight.copy_(0.1 * torch.randn(module.gate.weight.shape, generator=g))
    if module.route_bias is not None:
        module.route_bias.copy_(0.1 * torch.randn(module.route_bias.shape, generator=g))
    return module


@pytest.mark.parametrize("dtype,kw,head_dim,page", [
    (BF, dict(), 128, 16),
    (FP, dict(scoring="sigmoid", n_groups=4, topk_groups=2, route_scale=2.5, window=40, softcap=30.0), 64, 24)])
def test_steps(cuda, monkeypatch, dtype, kw, head_dim, page):
    dims, heads, kv_heads, experts, top_k, n = 512, 8, 2, 16, 4, 4
    layers = [fill(serve.PagedDecoderLayer(dims, heads, kv_heads, head_dim, experts, top_k, 256, "q4_k", "q6_k",
                                           dtype=dtype, device=cuda, **kw), s) for s in (1, 2)]
    cache = serve.PagedKVCache(2, 40, page, kv_heads, head_dim, n, dtype=dtype, device=cuda)
    cos, sin = serve.rope_tables(512, head_dim, device=cuda)
    calls = {}

    def record(name):
        fn = getattr(kq, name)

        def wrapped(*a, **k):
            r = fn(*a, **k)
            calls.setdefault(name, []).append((a, k, r))
            return r
        monkeypatch.setattr(kq, name, wrapped)

    for name in ("rope_kv_write", "paged_attention", "moe_route"):
        record(name)
    torch.manual_seed(0)
    u = U[dtype]
    sub = 2.0 ** -25 if dtype == FP else 0
    lens = [0] * n
    history = [[None] * n for _ in layers]  # (keys before their turn, values) of each request
    for step_no, new in enumerate([[130, 1, 0, 37], [1, 1, 64, 1], [1, 0, 1, 1], None, [1, 9, 1, 1]]):
        if new is None:  # a request ends and another takes its place and its pages
            cache.release(1)
            lens[1] = 0
            for h in history:
                h[1] = None
            continue
        calls.clear()
        step = cache.plan(new)
        x = torch.randn(sum(new), dims, device=cuda).to(dtype)
        pos = torch.cat([torch.arange(c, c + m, device=cuda) for c, m in zip(lens, new)])
        lens = [c + m for c, m in zip(lens, new)]
        cu = [sum(new[:i]) for i in range(n + 1)]
        for i, layer in enumerate(layers):
            y = layer(x, cos, sin, cache, i, step)
            (q, k, v, *_), _, turned = calls["rope_kv_write"][i]
            # rotation and cache contents, found through the tables
            ref, size = rope_ref(q, cos[pos], sin[pos], head_dim, False)
            assert ((turned.double() - ref).abs() <= u * ref.abs() + 2.0 ** -22 * size + sub).all()
            for b in range(n):
                rows = slice(cu[b], cu[b + 1])
                old = history[i][b]
                history[i][b] = (k[rows], v[rows]) if old is None else tuple(map(torch.cat, zip(old, (k[rows], v[rows]))))
                if not lens[b]:
                    continue
                at = torch.arange(lens[b], device=cuda)
                pages = cache.tables[b, at // page].long()
                kk, vv = history[i][b]
                ref, size = rope_ref(kk, cos[at], sin[at], head_dim, False)
                off = (cache.k[i][pages, at % page].double() - ref).abs()
                assert (off <= u * ref.abs() + 2.0 ** -22 * size + sub).all()
                assert torch.equal(cache.v[i][pages, at % page], vv)
            a, _, out = calls["paged_attention"][i]
            ref, _, tol, _ = attn_ref(turned, cache.k[i], cache.v[i], cache.tables, torch.tensor(lens),
                                      torch.tensor(cu), head_dim ** -0.5, layer.window, layer.softcap, True)
            assert ((out.double() - ref).abs() <= tol).all()
            (logits, *_), _, (idx, w) = calls["moe_route"][i]
            r = layer.routing
            ref_i, ref_w = route_ref(logits, top_k, r["scoring"] == "sigmoid", layer.route_bias, r["n_groups"],
                                     r["topk_groups"], True, r["scale"])
            assert torch.equal(idx.long(), ref_i) and ((w.double() - ref_w).abs() <= 2.0 ** -20 * ref_w.abs()).all()
            mid = x + layer.o(out.reshape(len(x), -1))
            normed = serve._rms_norm(mid, layer.ffn_norm, layer.eps)
            assert torch.equal(logits, layer.gate(normed))
            assert torch.equal(y, mid + layer.experts(normed, idx, w)) and torch.isfinite(y).all()
            x = y
        held = cache.tables[torch.arange(n, device=cuda)]
        used = torch.cat([held[b, :-(-lens[b] // page)] for b in range(n)] + [cache.free])
        assert sorted(used.tolist()) == list(range(40))  # every page once: in a table or free
    assert kq.workspace_error() == 0


def test_an_idle_step_changes_nothing(cuda):
    layer = fill(serve.PagedDecoderLayer(512, 8, 2, 64, 8, 2, 256, device=cuda), 3)
    cache = serve.PagedKVCache(1, 4, 16, 2, 64, 2, device=cuda)
    cos, sin = serve.rope_tables(64, 64, device=cuda)
    step = cache.plan([0, 0])
    x = torch.empty(0, 512, device=cuda, dtype=BF)
    assert layer(x, cos, sin, cache, 0, step).shape == (0, 512) and cache.lens == [0, 0]
    assert cache.k.count_nonzero() == 0 and kq.workspace_error() == 0
