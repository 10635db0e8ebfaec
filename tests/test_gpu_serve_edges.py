"""Edges of the serving-step operators.  Tolerances are those of
``test_gpu_serve_ops`` (derived there)."""
import pytest
import torch

from gmlx_b200 import kq, serve

from test_gpu_serve_ops import BF, FP, INF, attn_inputs, attn_ref, check_attn, i32, slow

pytestmark = pytest.mark.gpu


# A capped score is cap * tanh(score / cap), good to a few 2^-24 of the score, whatever the
# cap: below the f32 error of the score's own dot product, which the tolerance holds.
@pytest.mark.parametrize("softcap", [1e-3, 1.0, 1e3, 1e4, 1e5, 1e8, 3e38])
@pytest.mark.parametrize("lens,d,dtype", [([(1, 700), (3, 900)], 128, BF), ([(1, 700), (3, 900)], 64, FP),
                                          ([(130, 700), (1, 50)], 128, BF), ([(130, 700), (40, 300)], 64, FP),
                                          ([(130, 300)], 256, BF)])
def test_caps_far_from_the_scores(cuda, lens, d, dtype, softcap):
    check_attn(attn_inputs(cuda, lens, 8, 2, d, 16, dtype), max(n for n, _ in lens), softcap=softcap)


@pytest.mark.parametrize("what", ["cache heads", "cache rows", "cache pages", "query heads", "query tokens"])
@pytest.mark.parametrize("lens", [[(1, 200), (3, 40)], [(150, 400), (1, 77), (40, 40)], [(60, 200)]])
def test_expanded_tensors(cuda, lens, what):
    """Entries that stand at the same place (stride 0): one kv head shared by all by
    ``expand`` and the like, for chunks and single tokens alike."""
    q, kc, vc, *rest = attn_inputs(cuda, lens, 8, 4, 128, 16, BF)
    if what == "cache heads":
        kc, vc = (c[:, :, 1:2].expand(-1, -1, 4, -1) for c in (kc, vc))
    elif what == "cache rows":
        kc, vc = (c[:, 3:4].nan_to_num(0.5).expand(-1, 16, -1, -1) for c in (kc, vc))
    elif what == "cache pages":
        kc, vc = (c[2:3].nan_to_num(0.5).expand(c.shape[0], -1, -1, -1) for c in (kc, vc))
    elif what == "query heads":
        q = q[:, 2:3].expand(-1, 8, -1)
    else:
        q = q[1:2].expand(q.shape[0], -1, -1)
    assert 0 in (*q.stride(), *kc.stride())
    check_attn((q, kc, vc, *rest), max(n for n, _ in lens))


def test_expanded_heads_are_turned_and_stored(cuda):
    """Queries, keys and values of one head, expanded to several: as their copies."""
    q, k, v = (torch.randn(5, 1, 64, device=cuda).to(BF).expand(-1, h, -1) for h in (4, 2, 2))
    angle = torch.randn(8, 32, device=cuda)
    slots = torch.arange(5, device=cuda)
    outs = []
    for args in ((q, k, v), (q.contiguous(), k.contiguous(), v.contiguous())):
        kc, vc = torch.zeros(2, 2, 4, 2, 64, device=cuda, dtype=BF)
        outs.append((kq.rope_kv_write(*args, angle.cos(), angle.sin(), slots.int(), kc, vc, slots), kc, vc))
    assert all(torch.equal(a, b) for a, b in zip(*outs)) and kq.workspace_error() == 0


@pytest.mark.parametrize("max_q", [1, 1000])
@pytest.mark.parametrize("b,t,hq,hk,d,keys", [(1000, 1000, 32, 8, 128, 1024), (64, 8192, 32, 8, 64, 16384), (2, 7, 4, 2, 256, 64),
                                              (1500, 300, 8, 8, 64, 300)])
def test_descending_offsets_leave_every_row_empty(cuda, b, t, hq, hk, d, keys, max_q):
    """Requests that share tokens are far more work than the tokens there are: no request
    is computed, nothing is left behind in the workspace, and later calls are right."""
    valid = attn_inputs(cuda, [(1, 5000), (1, 40), (70, 900)], 8, 2, d, 16, BF)
    good = kq.paged_attention(*valid, 70, return_lse=True)
    q = torch.randn(t, hq, d, device=cuda).to(BF)
    kc, vc = torch.randn(2, 4, 64, hk, d, device=cuda).to(BF)
    table = torch.zeros(b, -(-keys // 64), dtype=torch.int32, device=cuda)
    for cu in ([0 if i % 2 == 0 else t for i in range(b + 1)], [0] + [t] * (b - 1) + [t - 1]):
        out, lse = kq.paged_attention(q, kc, vc, table, i32([keys] * b, cuda), i32(cu, cuda), max_q, return_lse=True)
        assert kq.workspace_error() == 20 and kq.workspace_error() == 0
        assert (out == 0).all() and (lse == -INF).all()
        key = (torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)
        ws = kq._ext().workspace_peek(*key) if kq._ext() is not None else kq._WS[key]
        assert not ws[256:256 + (1 << 20)].any()  # the counters (in front, the group count of an expert call may stand)
        again = kq.paged_attention(*valid, 70, return_lse=True)
        assert torch.equal(again[0], good[0]) and torch.equal(again[1], good[1])
    assert kq.workspace_error() == 0


@pytest.mark.parametrize("d,dtype", [(64, FP), (128, BF), (256, BF)])
@pytest.mark.parametrize("lens", [[(1, 5000), (1, 30)], [(150, 5000), (40, 40)]])
def test_nan_reaches_its_rows_and_no_others(cuda, lens, d, dtype):
    """A NaN query, and a NaN key in the last position of a request (one row sees it):
    those rows are NaN, sum and output, however the row is split; the others are as without."""
    args = attn_inputs(cuda, lens, 4, 2, d, 16, dtype)
    ref, ref_l, tol, tol_l = attn_ref(*args, d ** -0.5, 0, 0.0, True)
    q, kc = args[0].clone(), args[1].clone()
    q[0, 1, 3] = float("nan")
    last = lens[0][1] - 1
    kc[args[3][0, last // 16].long(), last % 16, 1, 5] = float("nan")  # kv head 1: query heads 2 and 3
    out, lse = kq.paged_attention(q, kc, *args[2:], max(n for n, _ in lens), return_lse=True)
    hit = torch.zeros(lse.shape, dtype=torch.bool, device=cuda)
    hit[0, 1] = True
    hit[lens[0][0] - 1, 2:] = True
    assert lse[hit].isnan().all() and out[hit].isnan().all()
    assert ((out.double() - ref).abs() <= tol)[~hit].all() and ((lse.double() - ref_l).abs() <= tol_l)[~hit].all()
    assert kq.workspace_error() == 0


def fresh_stream(cuda):
    """A stream that no call has used (handles of destroyed streams may come again)."""
    for _ in range(64):
        s = torch.cuda.Stream()
        key = (torch.cuda.current_device(), s.cuda_stream)
        e = kq._ext()
        if (e.workspace_peek(*key) is None if e is not None else True) and key not in kq._WS:
            return s
    pytest.skip("no unused stream")


def overdrawn_plan(cuda):
    kq.paged_plan(i32([0], cuda), i32([4], cuda), i32([[-1]], cuda), i32([], cuda), 4, 4)


@pytest.mark.parametrize("call", [lambda f, *a: f(*a), slow], ids=["native", "python"])
def test_a_growing_workspace_keeps_its_error_word(cuda, call):
    """The plan's missing page is still reported after the stream's first attention."""
    args = attn_inputs(cuda, [(2, 30)], 4, 2, 64, 16, BF)
    s = fresh_stream(cuda)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(overdrawn_plan, cuda)
        call(kq.paged_attention, *args, 2)
        assert call(kq.workspace_error) == 21 and call(kq.workspace_error) == 0


@pytest.mark.parametrize("call", [lambda f, *a: f(*a), slow], ids=["native", "python"])
def test_a_captured_workspace_outlives_its_growth(cuda, call):
    """A graph keeps the workspace it was captured with, to itself, and errors that its
    replays record there are seen."""
    small = attn_inputs(cuda, [(1, 900)], 4, 2, 64, 16, BF)
    large = attn_inputs(cuda, [(1, 900)], 4, 2, 256, 16, BF)
    seq = small[4].clone()
    s = fresh_stream(cuda)
    s.wait_stream(torch.cuda.current_stream())
    key = (torch.cuda.current_device(), s.cuda_stream)

    def workspace():
        return kq._ext().workspace_peek(*key) if kq._EXT else kq._WS[key]

    with torch.cuda.stream(s):
        ref = call(kq.paged_attention, *small, 1)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = call(kq.paged_attention, *small[:4], seq, small[5], 1)
    with torch.cuda.stream(s):
        old = call(workspace)
        lo, size = old.data_ptr(), old.numel()
        del old
        call(kq.paged_attention, *large, 1)
        assert call(workspace).data_ptr() != lo
        # what the caching allocator hands out now must not be the graph's workspace
        others = [torch.full((size,), 255, dtype=torch.uint8, device=cuda) for _ in range(4)]
        assert all(t.data_ptr() + size <= lo or lo + size <= t.data_ptr() for t in others)
        g.replay()
        assert torch.equal(out, ref) and all((t == 255).all() for t in others)
        assert call(kq.workspace_error) == 0
        seq.fill_(10 ** 6)
        g.replay()
        assert call(kq.workspace_error) == 20 and call(kq.workspace_error) == 0


def test_a_step_does_not_wait_for_the_device(cuda):
    layer = serve.PagedDecoderLayer(512, 8, 2, 64, 8, 2, 256, device=cuda)
    cache = serve.PagedKVCache(1, 16, 16, 2, 64, 2, device=cuda)
    cos, sin = serve.rope_tables(256, 64, device=cuda)
    x = torch.zeros(6, 512, device=cuda, dtype=BF)
    layer(x, cos, sin, cache, 0, cache.plan([5, 1]))  # kernels are loaded, workspaces made
    torch.cuda.set_sync_debug_mode("error")
    try:
        step = cache.plan([1, 5])
        layer(x, cos, sin, cache, 0, step)
        cache.release(0)
        cache.plan([3, 0])
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert step.plan.seq_lens.tolist() == [6, 6] and kq.workspace_error() == 0


def test_lengths_of_many_steps_in_flight(cuda):
    """Plans that are queued faster than the device takes them: each sees its own lengths."""
    cache = serve.PagedKVCache(1, 64, 16, 1, 64, 3, device=cuda)
    a = torch.randn(4096, 4096, device=cuda)
    torch.cuda.synchronize()
    for _ in range(20):  # the device is busy for some milliseconds
        a = a @ a * 1e-2
    steps = [cache.plan([i % 3, 1, 0]) for i in range(100)]
    lens = [0, 0, 0]
    for i, s in enumerate(steps):
        lens = [lens[0] + i % 3, lens[1] + 1, 0]
        assert s.plan.seq_lens.tolist() == lens
    assert kq.workspace_error() == 0


@pytest.mark.parametrize("e,groups", [(64, 8), (512, 4)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_stays_in_the_open_groups(cuda, e, groups, scoring):
    """Experts that the bias rules out (-inf), so that fewer than k are left in the open
    groups: the rest of the choice are the ruled-out ones there, lowest first."""
    size, k = e // groups, 8
    first = e - 2 * size
    logits = torch.randn(33, e, device=cuda)
    bias = torch.full((e,), -10.0, device=cuda)
    bias[first:] = -INF
    left = [first + 2, first + 3, e - 3, e - 2]  # two of each of the last two groups, which rank highest
    bias[left] = 0.0
    idx, w = kq.moe_route(logits, k, scoring, bias, groups, 2)
    rest = [i for i in range(first, e) if i not in left][:k - 4]
    assert all(set(r[:4]) == set(left) and r[4:] == rest for r in idx.tolist())
    assert torch.isfinite(w).all()


@pytest.mark.parametrize("call", [lambda f, *a: f(*a), slow], ids=["native", "python"])
def test_a_workspace_made_in_a_capture_is_none_of_the_graph_s_work(cuda, call):
    """Two graphs of a stream that no call has used before: either may run first, and
    neither's replay wipes what the other recorded."""
    args = attn_inputs(cuda, [(1, 900), (2, 300)], 8, 2, 64, 16, BF)
    plan = (i32([0], cuda), i32([4], cuda), i32([[-1]], cuda), i32([7], cuda), 4, 4)
    ref = kq.paged_attention(*args, 2)
    seq = args[4].clone()
    s = fresh_stream(cuda)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            if not graphs:
                call(kq.paged_plan, *plan)  # a small workspace, which the attention outgrows
            outs.append(call(kq.paged_attention, *args[:4], seq, args[5], 2))
        graphs.append(g)
    key = (torch.cuda.current_device(), s.cuda_stream)
    ws = kq._ext().workspace_peek(*key) if kq._EXT and call is not slow else kq._WS[key]
    assert not ws.any()
    with torch.cuda.stream(s):
        graphs[1].replay()
        assert torch.equal(outs[1], ref) and call(kq.workspace_error) == 0
        seq.fill_(10 ** 6)
        graphs[1].replay()
        seq.copy_(args[4])
        graphs[0].replay()
        assert torch.equal(outs[0], ref)
        assert call(kq.workspace_error) == 20 and call(kq.workspace_error) == 0
        graphs[1].replay()
        assert torch.equal(outs[1], ref) and call(kq.workspace_error) == 0
