"""What the serving-step operators and their step decide on the host: argument
checks of the C entries (answered before any CUDA call), refusals of tensors that
are not on a GPU, and the page accounting of the cache."""
import ctypes

import pytest
import torch

from gmlx_b200 import _lib, build, kq, serve

P = 16  # stands for a device pointer: 16-byte aligned, never followed here


def cache(**kw):
    c = dict(k=P, v=P, dtype=_lib.KQ_BF16, pages=4, page_size=16, kv_heads=2, dim=128, page_stride=16 * 256,
             row_stride=256, head_stride=128)
    c.update(kw)
    return ctypes.byref(_lib.PagedCache(*c.values()))


def call(name, defaults, **kw):
    args = dict(defaults, **kw)
    return getattr(_lib.load(), name)(*args.values())


PLAN = dict(ctx=P, new=P, batch=2, tables=P, stride=4, width=4, free=P, n_free=4, page=16, tokens=8, cu=P, seq=P,
            slots=P, pos=P, used=P, ws=P, ws_bytes=256, stream=None)
ROPE = dict(cache=None, q=P, qt=512, qh=128, k=P, kt=256, kh=128, v=P, vt=256, vh=128, tokens=2, heads=4, cos=P, sin=P,
            n_pos=8, rot=128, inter=0, pos=P, slots=P, out=P, ws=P, ws_bytes=256, stream=None)
ATTN = dict(cache=None, q=P, qt=512, qh=128, tokens=2, heads=4, tables=P, stride=4, width=4, seq=P, cu=P, batch=1,
            max_q=2, scale=0.1, causal=1, window=0, softcap=0.0, out=P, lse=None, ws=P, ws_bytes=1 << 40, stream=None)
ROUTE = dict(logits=P, dtype=_lib.KQ_F32, t=2, e=64, stride=64, k=4, scoring=0, bias=None, groups=1, top=1, norm=1,
             scale=1.0, idx=P, w=P, stream=None)


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(batch=8193), dict(page=0), dict(tokens=-1), dict(width=-1),
                                dict(stride=3), dict(n_free=-1)])
def test_plan_shapes(kw):
    assert call("kq_paged_plan", PLAN, **kw) == _lib.KQ_ERR_SHAPE
    assert b"paged_plan" in _lib.load().kq_last_error()


@pytest.mark.parametrize("kw", [dict(heads=-1), dict(tokens=-1), dict(rot=8), dict(rot=144), dict(n_pos=0),
                                dict(cache=dict(dim=24)), dict(cache=dict(pages=0)), dict(cache=dict(k=0))])
def test_rope_shapes(kw):
    kw = dict(kw, cache=cache(**kw.get("cache", {})))
    assert call("kq_rope_kv_write", ROPE, **kw) == _lib.KQ_ERR_SHAPE
    assert b"rope_kv_write" in _lib.load().kq_last_error()


@pytest.mark.parametrize("kw", [dict(heads=3), dict(tokens=-1), dict(scale=0.0), dict(scale=float("nan")),
                                dict(window=-1), dict(window=5, causal=0), dict(softcap=-1.0),
                                dict(cache=dict(dim=96)), dict(batch=-1), dict(stride=3)])
def test_attention_shapes(kw):
    kw = dict(kw, cache=cache(**kw.get("cache", {})))
    assert call("kq_paged_attention", ATTN, **kw) == _lib.KQ_ERR_SHAPE
    assert b"paged_attention" in _lib.load().kq_last_error()


@pytest.mark.parametrize("kw", [dict(e=1025), dict(e=0), dict(k=0), dict(k=33), dict(e=8, k=9), dict(groups=5),
                                dict(groups=64), dict(groups=4, top=5), dict(groups=4, top=0), dict(scoring=2),
                                dict(scale=float("inf")), dict(t=-1)])
def test_route_shapes(kw):
    assert call("kq_moe_route", ROUTE, **kw) == _lib.KQ_ERR_SHAPE
    assert b"moe_route" in _lib.load().kq_last_error()


@pytest.mark.parametrize("kw", [dict(qt=516), dict(q=8), dict(cache=dict(row_stride=252)), dict(cache=dict(v=8)),
                                dict(out=8)])
def test_alignment(kw):
    kw = dict(kw, cache=cache(**kw.get("cache", {})))
    assert call("kq_rope_kv_write", ROPE, **kw) == _lib.KQ_ERR_ALIGN
    assert call("kq_paged_attention", ATTN, **kw) == _lib.KQ_ERR_ALIGN


def test_workspaces():
    for name, args in (("kq_paged_plan", PLAN), ("kq_rope_kv_write", dict(ROPE, cache=cache())),
                       ("kq_paged_attention", dict(ATTN, cache=cache()))):
        assert call(name, args, ws_bytes=255) == _lib.KQ_ERR_WORKSPACE
        assert call(name, args, ws=None) == _lib.KQ_ERR_WORKSPACE


def test_types():
    assert call("kq_rope_kv_write", ROPE, cache=cache(dtype=_lib.KQ_F32)) == _lib.KQ_ERR_DTYPE
    assert call("kq_paged_attention", ATTN, cache=cache(dtype=_lib.KQ_F32)) == _lib.KQ_ERR_DTYPE
    assert call("kq_moe_route", ROUTE, dtype=9) == _lib.KQ_ERR_DTYPE


def test_ops_refuse_tensors_outside_the_gpu():
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    c = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    a = torch.zeros(4, 32)
    with pytest.raises(ValueError, match="CUDA"):
        kq.paged_plan(i, i, i.view(1, 1), i, 4, 1)
    with pytest.raises(ValueError, match="CUDA"):
        kq.rope_kv_write(x, x, x, a, a, i, c, c, i.long())
    with pytest.raises(ValueError, match="CUDA"):
        kq.paged_attention(x, c, c, i.view(1, 1), i, torch.zeros(2, dtype=torch.int32), 1)
    with pytest.raises(ValueError, match="CUDA"):
        kq.moe_route(torch.zeros(2, 8), 2)
    with pytest.raises(ValueError, match="scoring"):
        kq.moe_route(torch.zeros(2, 8), 2, "relu")


def test_extension_exports_the_serving_ops():
    mod = build.load_torch_ext()
    if mod is None:
        pytest.skip("gmlx_b200/_ext/kq_torch.so not built")
    for name in ("set_serve_entry_points", "paged_plan", "rope_kv_write", "paged_attention", "moe_route"):
        assert hasattr(mod, name)


def test_cache_accounting(monkeypatch):
    """Pages are counted on the host as the plan hands them out on the GPU."""
    seen = []
    monkeypatch.setattr(kq, "paged_plan", lambda *a: seen.append(a))
    c = serve.PagedKVCache(1, 6, 4, 1, 64, 3, max_pages=4)
    s = c.plan([5, 0, 4])
    ctx, new, tables, free, page, tokens = seen[0]
    assert (ctx.tolist(), new.tolist(), page, tokens, s.max_query_len) == ([0, 0, 0], [5, 0, 4], 4, 9, 5)
    assert tables is c.tables and free.tolist() == list(range(6))
    assert c.lens == [5, 0, 4] and c.free.tolist() == [3, 4, 5]
    c.tables[0, :2] = torch.tensor([0, 1])
    c.plan([3, 1, 1])  # fills request 0's page, takes one each for the others
    assert seen[1][0].tolist() == [5, 0, 4] and c.free.tolist() == [5]
    for bad, why in (([1, 3, 4], "free"), ([9, 0, 0], "more than 4"), ([1, 1], "lengths"), ([0, 0, -1], "lengths")):
        with pytest.raises(ValueError, match=why):
            c.plan(bad)
    assert c.lens == [8, 1, 5] and len(seen) == 2
    c.release(0)
    assert c.lens == [0, 1, 5] and c.free.tolist() == [5, 0, 1]
    c.plan([0, 0, 0])
    assert seen[2][5] == 0


def test_rope_tables():
    cos, sin = serve.rope_tables(70000, 64, 1e6)
    assert cos.shape == sin.shape == (70000, 32) and cos.dtype == torch.float32
    a = 69999 * 1e6 ** (-2 * 5 / 64)
    assert abs(float(cos[69999, 5]) - torch.tensor(a, dtype=torch.float64).cos().item()) <= 2.0 ** -24
    assert (cos[0] == 1).all() and (sin[0] == 0).all()
