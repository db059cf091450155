"""Token-level operators in the calls around the ordinary ones: lengths and
sums that the kernel before writes and the kernel after reads, several streams,
threads and graphs at once, batches and head groups beyond the usual, caches
without capacity, tables with pages named twice.  Bounds: ``token_ref``."""
import math
import threading

import pytest
import torch

import token_ref as R

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=BF):
    return torch.randn(shape, generator=g).to(dtype).cuda()


def _qkv(g, B, N, Hq, Hkv, S, D, dtype=BF):
    return (_randn(g, B, N, Hq, D, dtype=dtype), _randn(g, B, S, Hkv, D, dtype=dtype),
            _randn(g, B, S, Hkv, D, dtype=dtype))


@pytest.mark.parametrize("N,S", [(1, 700), (40, 700), (40, 5000)])
def test_neighbours_on_the_stream(N, S):
    """A captured chain: the lengths are written right before a call and its
    results read right after it, with keys that fit one run and many."""
    import orthocache_b200 as oc
    g = _gen(1)
    B, Hq, Hkv, D = 3, 8, 2, 128
    q, k, v = _qkv(g, B, N, Hq, Hkv, S, D)
    start = torch.tensor([S - 90, S // 2, 60], dtype=torch.int32, device="cuda")
    lens, step = start.clone(), torch.full((B,), 9, dtype=torch.int32, device="cuda")
    w = torch.zeros(B, Hkv, S, device="cuda")
    outs = [torch.empty_like(q) for _ in range(8)]
    sums = torch.empty(8, B, Hkv, S, device="cuda")

    def chain():
        for i in range(8):
            lens.add_(step)
            if i % 2:
                o, nw = oc.accumulate_attention(q, k, v, w, lens, out_weights=w)
            else:
                o, nw = oc.chunk_attention(q, k, v, lens), w
            outs[i].copy_(o)
            sums[i].copy_(nw)

    chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    for _ in range(3):
        lens.copy_(start)
        w.zero_()
        graph.replay()
    got, got_sums = [o.clone() for o in outs], sums.clone()
    w0 = torch.zeros_like(w)
    for i in range(8):
        n = start + (i + 1) * step
        torch.cuda.synchronize()
        if i % 2:
            want, w0 = oc.accumulate_attention(q, k, v, w0, n)
        else:
            want = oc.chunk_attention(q, k, v, n)
        torch.cuda.synchronize()
        assert torch.equal(got[i], want), i
        assert torch.equal(got_sums[i], w0), i


def test_graphs_and_streams_at_once():
    """Two captured graphs and two eager streams in flight together: nothing they
    use is shared."""
    import orthocache_b200 as oc
    g = _gen(2)
    B, Hq, Hkv, S, D = 2, 16, 4, 3000, 128
    lens = torch.tensor([S, 1900], dtype=torch.int32, device="cuda")
    sets = [(_qkv(g, B, n, Hq, Hkv, S, D)) for n in (1, 130, 5, 70)]
    w = torch.rand(B, Hkv, S, generator=g).cuda()
    mask = torch.stack([R.random_tree(70, g) for _ in range(B)]).cuda()
    dk, dv = _randn(g, B, 70, Hkv, D), _randn(g, B, 70, Hkv, D)

    def ops():
        return [lambda: oc.accumulate_attention(*sets[0], w, lens)[1],
                lambda: oc.chunk_attention(*sets[1], lens, cap=30.0),
                lambda: oc.chunk_attention(*sets[2], lens),
                lambda: oc.tree_attention(sets[3][0], sets[3][1], sets[3][2], dk, dv, mask, lens)]

    want = [f() for f in ops()]
    torch.cuda.synchronize()
    graphs, held = [], []
    for f in ops()[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(f())
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                if i < 2:
                    graphs[i].replay()
                    got.append((i, held[i].clone()))
                else:
                    got.append((i, ops()[i]()))
    torch.cuda.synchronize()
    for i, x in got:
        assert torch.equal(x, want[i]), i


def test_threads_at_once():
    import orthocache_b200 as oc
    g = _gen(3)
    cases = [_qkv(g, 1, n, 8, 2, 900, d, t) for n, d, t in ((3, 64, F32), (40, 256, BF), (130, 64, BF), (2, 256, F32))]
    want = [oc.chunk_attention(*c, cap=20.0) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got = oc.chunk_attention(*cases[i], cap=20.0)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[i]):
                    bad.append(i)
        except Exception as e:  # reported below, by the main thread
            bad.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,N,Hq,Hkv,S,D", [
    (300, 1, 4, 2, 70, 64),     # more batch rows than the even cut adds up
    (300, 40, 4, 2, 130, 64),
    (1, 1, 256, 1, 300, 128),   # one KV head for all
    (1, 3, 130, 1, 200, 64),
    (2, 9, 35, 5, 333, 128),    # odd groups of heads
    (1, 50, 11, 1, 260, 256),
    (2, 300, 2, 2, 100, 64),    # a chunk longer than the capacity
])
def test_batches_and_heads(B, N, Hq, Hkv, S, D, dtype):
    import orthocache_b200 as oc
    g = _gen(B + N + Hq)
    q, k, v = _qkv(g, B, N, Hq, Hkv, S, D, dtype)
    lengths = [max(0, S - 7 * (b % 11)) for b in range(B)]
    vis = R.chunk_visible(lengths, N, S).cuda()
    kd, vd = k.clone(), v.clone()
    for b, n in enumerate(lengths):
        kd[b, n:] = math.nan
        vd[b, n:] = math.nan
    w0 = torch.rand(B, Hkv, S, generator=g).cuda()
    out, sums = oc.accumulate_attention(q, kd, vd, w0, torch.tensor(lengths))
    want, p, tol, rel = R.attend(q, kd, vd, vis)
    R.check(out, want, tol)
    p = torch.where(vis.any(2)[:, None, :, None], p, torch.zeros_like(p))
    ws, wtol = R.column_sums(p, rel, Hkv)
    R.check(sums, w0.double() + ws, wtol + 2.0 ** -24 * (w0.double() + ws))  # and the last addition


def test_more_heads_than_a_grid_has_rows():
    import orthocache_b200 as oc
    g = _gen(4)
    B, H, S, D = 1100, 64, 5, 64
    q, k, v = _qkv(g, B, 1, H, H, S, D)
    out, sums = oc.accumulate_attention(q, k, v)
    want, p, tol, rel = R.attend(q, k, v, torch.ones(B, 1, S, dtype=torch.bool, device="cuda"))
    R.check(out, want, tol)
    ws, wtol = R.column_sums(p, rel, H)
    R.check(sums, ws, wtol + 2.0 ** -24 * ws)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,D", [(1, 64), (80, 128), (80, 256)])
def test_no_capacity(N, D, dtype):
    import orthocache_b200 as oc
    g = _gen(5)
    q, k, v = _qkv(g, 2, N, 4, 2, 0, D, dtype)
    assert not oc.chunk_attention(q, k, v).any()
    assert not oc.chunk_attention(q, k, v, documents=torch.zeros(2, 0, dtype=torch.int32), cap=3.0).any()
    out, sums = oc.accumulate_attention(q, k, v)
    assert not out.any() and sums.shape == (2, 2, 0)
    cache = oc.PagedKVCache(2, 2, D, dtype=dtype)
    dk, dv = _randn(g, 2, N, 2, D, dtype=dtype), _randn(g, 2, N, 2, D, dtype=dtype)
    mask = R.random_tree(N, g)
    out = cache.attend_tree(q, dk, dv, mask.cuda(), torch.zeros(2, 0, dtype=torch.int32), torch.tensor([0, 5]))
    want, _, tol, _ = R.attend(q, dk, dv, mask.expand(2, N, N).cuda())
    R.check(out, want, tol)


@pytest.mark.parametrize("dtype,T", [(BF, 2), (BF, 90), (F32, 3)])
def test_a_page_named_twice(dtype, T):
    import orthocache_b200 as oc
    g = _gen(6)
    Hq, Hkv, D = 4, 2, 128
    cache = oc.PagedKVCache(3, Hkv, D, dtype=dtype)
    cache.k.copy_(_randn(g, *cache.k.shape, dtype=dtype))
    cache.v.copy_(_randn(g, *cache.v.shape, dtype=dtype))
    table = torch.tensor([[2, 0, 2], [2, 2 ** 31 + 1, 1]])  # int64; the second row's middle page is outside the pool
    q, dk, dv = (_randn(g, 2, T, h, D, dtype=dtype) for h in (Hq, Hkv, Hkv))
    mask = R.random_tree(T, g)
    lens = torch.tensor([1300, 2 ** 32 + 9])  # beyond int32: all of the capacity
    out = cache.attend_tree(q, dk, dv, mask.cuda(), table, lens)
    pool_k, pool_v = (x.view(3, 512, Hkv, D) for x in (cache.k, cache.v))
    idx = torch.tensor([[2, 0, 2], [2, 0, 1]], device="cuda")
    k, v = pool_k[idx].reshape(2, 1536, Hkv, D), pool_v[idx].reshape(2, 1536, Hkv, D)
    past = torch.ones(2, 1536, dtype=torch.bool)
    past[0, 1300:] = False
    past[1, 512:1024] = False
    vis = torch.cat([past[:, None].expand(2, T, 1536), mask.expand(2, T, T)], 2).cuda()
    want, _, tol, _ = R.attend(q, torch.cat([k, dk], 1), torch.cat([v, dv], 1), vis)
    R.check(out, want, tol)


@pytest.mark.parametrize("N", [1, 40, 200])
@pytest.mark.parametrize("cap,scale", [(0.01, 0.5), (1e-4, 0.4), (300.0, 9.0), (2.0, -0.3)])
def test_caps_from_far_below_the_scores_to_above(N, cap, scale):
    import orthocache_b200 as oc
    g = _gen(7)
    q, k, v = _qkv(g, 1, N, 4, 2, 400, 128)
    q[:, :, 0] = 0  # scores of zero too
    vis = R.chunk_visible([390], N, 400).cuda()
    out, sums = oc.accumulate_attention(q, k, v, None, 390, cap=cap, scale=scale)
    want, p, tol, rel = R.attend(q, k, v, vis, cap=cap, scale=scale)
    R.check(out, want, tol)
    ws, wtol = R.column_sums(p, rel, 2)
    R.check(sums, ws, wtol)


def test_caps_and_sums_refused():
    import orthocache_b200 as oc
    g = _gen(8)
    q, k, v = _qkv(g, 1, 2, 4, 2, 64, 64)
    for cap, scale in ((1e-30, None), (1e-60, None), (1e-5, -0.1), (1e6, 1e8)):
        with pytest.raises(ValueError, match="cap"):
            oc.chunk_attention(q, k, v, cap=cap, scale=scale)
    buf = torch.zeros(2 * 64 + 3, device="cuda")
    w, o = buf[:128].view(1, 2, 64), buf[3:].view(1, 2, 64)
    with pytest.raises(oc._lib.OrthoCacheError, match="overlap"):
        oc.accumulate_attention(q, k, v, w, out_weights=o)
    assert not buf.any()


@pytest.mark.parametrize("N,dtype", [(2, BF), (100, BF), (3, F32)])
def test_memory_around_the_results_is_left_alone(N, dtype):
    """Through the C interface, with guards before and behind every result and the workspace."""
    import orthocache_b200 as oc
    from orthocache_b200 import _lib
    g = _gen(9)
    B, Hq, Hkv, S, D = 2, 6, 2, 777, 128
    q, k, v = _qkv(g, B, N, Hq, Hkv, S, D, dtype)
    lens = torch.tensor([777, 5], dtype=torch.int32, device="cuda")
    code = _lib.dtype_code(k)
    ws_n = _lib.query("oc_token_attention_workspace_bytes", code, B, N, Hq, Hkv, D, S, 1)
    pad = 256

    def guarded(nbytes):
        t = torch.full((nbytes + 2 * pad,), 0xA5, dtype=torch.uint8, device="cuda")
        return t, t[pad:pad + nbytes]

    out_all, out = guarded(q.numel() * q.element_size())
    w_all, w = guarded(B * Hkv * S * 4)
    ws_all, ws = guarded(ws_n)
    assert ws_n > 0
    _lib.call("oc_accumulate_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), code, lens.data_ptr(), None,
              w.data_ptr(), B, N, Hq, Hkv, D, S, 0.0, 0.1, out.data_ptr(), code, ws.data_ptr(), ws_n,
              _lib.stream_ptr(k.device))
    torch.cuda.synchronize()
    for t in (out_all, w_all, ws_all):
        assert (t[:pad] == 0xA5).all() and (t[-pad:] == 0xA5).all()
    want, sums = oc.accumulate_attention(q, k, v, None, lens, scale=0.1)
    assert torch.equal(out.view(dtype).view_as(q), want)
    assert torch.equal(w.view(F32).view(B, Hkv, S), sums)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("N,G", [(3, 1), (1, 8), (4, 3), (8, 3), (6, 5), (31, 1)])
def test_few_rows_with_every_mask(N, G, D, dtype):
    """3 to 31 rows per KV head: a ragged batch with padding, documents, a prefix,
    a bias and a cap together, and the sums; keys enough for many runs."""
    import orthocache_b200 as oc
    g = _gen(N + G)
    B, Hkv, S = 3, 2, 1301
    Hq = Hkv * G
    q, k, v = _qkv(g, B, N, Hq, Hkv, S, D, dtype)
    lengths, prefix = [1301, 640, N], [900, 0, 2]
    docs = (torch.arange(S) // 450).int().repeat(B, 1)
    docs[0, 700:760] = -1
    docs[1, 100:400] = -1
    docs[1, :100] = 1
    kd, vd = k.clone(), v.clone()
    for b, n in enumerate(lengths):
        hidden = (torch.arange(S) >= n) | (docs[b] < 0)
        kd[b, hidden] = math.nan
        vd[b, hidden] = math.inf
    lens, slopes = torch.tensor(lengths), torch.linspace(0.001, 0.02, Hq)
    for kw in (dict(), dict(documents=docs), dict(documents=docs, prefix=prefix, slopes=slopes, cap=8.0)):
        if kw:
            vis = R.chunk_visible(lengths, N, S, prefix=kw.get("prefix"), documents=docs).cuda()
            ins = (q, kd, vd)
        else:
            vis = R.chunk_visible(lengths, N, S).cuda()
            ins = (q, k, v)
        bias = R.distance_bias(lengths, N, S, slopes).cuda() if "slopes" in kw else None
        args = {**kw, **({"prefix": torch.tensor(prefix)} if "prefix" in kw else {})}
        out = oc.chunk_attention(*ins, lens, **args)
        kz, vz = (torch.where(torch.isfinite(x), x, torch.zeros_like(x)) for x in ins[1:])
        want, p, tol, rel = R.attend(q, kz, vz, vis, cap=kw.get("cap", 0.0), bias=bias)
        R.check(out, want, tol, str(list(kw)))
        if not kw:
            out, sums = oc.accumulate_attention(*ins, None, lens)
            R.check(out, want, tol)
            ws, wtol = R.column_sums(p, rel, Hkv)
            R.check(sums, ws, wtol)
