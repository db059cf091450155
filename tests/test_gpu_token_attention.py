"""Token-level attention (tree, chunk, accumulating) against a float64
reference, at the sizes, masks and layouts where it can go wrong; the bounds
are those of ``token_ref``."""
import math

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


def _qkv(g, B, N, Hq, Hkv, S, D, dtype):
    q = _randn(g, B, N, Hq, D, dtype=dtype)
    k, v = _randn(g, B, S, Hkv, D, dtype=dtype), _randn(g, B, S, Hkv, D, dtype=dtype)
    if S:
        k[:, :: 17] += 0.5 * q[:, :1, :: Hq // Hkv]  # some keys stand out
    return q, k, v


def _dirty(k, v, lengths):
    """Poison what lies behind every sequence."""
    k, v = k.clone(), v.clone()
    for b, n in enumerate(lengths):
        k[b, max(n, 0):] = math.nan
        v[b, max(n, 0):] = math.inf
    return k, v


# ---------------------------------------------------------------------------
# tree
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,T,Hq,Hkv,S,D,cap", [
    (1, 1, 1, 1, 1, 64, 0.0),
    (1, 1, 32, 8, 600, 128, 0.0),
    (2, 5, 6, 2, 63, 64, 0.0),
    (2, 7, 8, 8, 130, 128, 20.0),
    (1, 16, 32, 8, 2049, 128, 0.0),
    (3, 33, 12, 4, 517, 128, 30.0),
    (1, 64, 7, 1, 1000, 64, 0.0),
    (2, 61, 32, 8, 1537, 128, 30.0),
    (2, 8, 32, 16, 777, 256, 0.0),
    (1, 100, 6, 2, 300, 256, 5.0),
    (1, 256, 4, 2, 40, 128, 0.0),
])
def test_tree_against_float64(B, T, Hq, Hkv, S, D, cap, dtype):
    import orthocache_b200 as oc
    g = _gen(B * 1000 + T * 10 + S)
    q, k, v = _qkv(g, B, T, Hq, Hkv, S, D, dtype)
    dk, dv = _randn(g, B, T, Hkv, D, dtype=dtype), _randn(g, B, T, Hkv, D, dtype=dtype)
    lengths = [max(0, S - 37 * b) for b in range(B)]
    mask = torch.stack([R.random_tree(T, g) for _ in range(B)])
    kd, vd = _dirty(k, v, lengths)
    out = oc.tree_attention(q, kd, vd, dk, dv, mask.cuda(), torch.tensor(lengths), cap=cap)
    vis = torch.cat([(torch.arange(S)[None] < torch.tensor(lengths)[:, None])[:, None].expand(B, T, S), mask], 2)
    want, _, tol, _ = R.attend(q, torch.cat([kd, dk], 1), torch.cat([vd, dv], 1), vis.cuda(), cap=cap)
    assert out.dtype == dtype
    R.check(out, want, tol)


@pytest.mark.parametrize("dtype,D,T", [(BF, 128, 3), (BF, 128, 40), (BF, 64, 9), (F32, 128, 5), (BF, 256, 6)])
def test_paged_tree(dtype, D, T):
    """Pages in any order, a last page that ends inside a tile, sequences of no
    page, table entries outside the pool, and unwritten (NaN) memory behind
    every sequence."""
    import orthocache_b200 as oc
    g = _gen(5 + T)
    lengths, Hq, Hkv, nb, pages = [1300, 512, 0, 1, 700], 8, 2, 3, 11
    B = len(lengths)
    q, k, v = _qkv(g, B, T, Hq, Hkv, nb * 512, D, dtype)
    dk, dv = _randn(g, B, T, Hkv, D, dtype=dtype), _randn(g, B, T, Hkv, D, dtype=dtype)
    cache = oc.PagedKVCache(pages, Hkv, D, dtype=dtype)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    free = torch.randperm(pages, generator=g).tolist()
    table = torch.full((B, nb), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        for j in range((n + 511) // 512):
            p = free.pop()
            table[b, j] = p
            m = min(512, n - 512 * j)
            cache.k.view(pages, 512, Hkv, D)[p, :m] = k[b, 512 * j:512 * j + m]
            cache.v.view(pages, 512, Hkv, D)[p, :m] = v[b, 512 * j:512 * j + m]
    hole = torch.ones(B, nb * 512, dtype=torch.bool)
    table[4, 0] = pages + 3  # outside the pool: nobody sees its tokens
    hole[4, :512] = False
    mask = R.random_tree(T, g)  # one mask for the whole batch
    out = cache.attend_tree(q, dk, dv, mask.cuda(), table, torch.tensor(lengths))
    past = (torch.arange(nb * 512)[None] < torch.tensor(lengths)[:, None]) & hole
    vis = torch.cat([past[:, None].expand(B, T, nb * 512), mask.expand(B, T, T)], 2).cuda()
    want, _, tol, _ = R.attend(q, torch.cat([k, dk], 1), torch.cat([v, dv], 1), vis)
    R.check(out, want, tol)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [4, 48])
def test_padded_tree_and_empty_rows(T, dtype):
    """A padded node sees nothing and is seen by nobody; over an empty cache its
    row is zero, whatever its keys and values hold."""
    import orthocache_b200 as oc
    g = _gen(T)
    B, Hq, Hkv, S, D = 2, 8, 2, 128, 128
    q, k, v = _qkv(g, B, T, Hq, Hkv, S, D, dtype)
    dk, dv = _randn(g, B, T, Hkv, D, dtype=dtype), _randn(g, B, T, Hkv, D, dtype=dtype)
    mask = torch.stack([R.random_tree(T, g) for _ in range(B)])
    mask[:, -2:] = False
    mask[:, :, -2:] = False
    dk[:, -2:] = math.nan
    dv[:, -2:] = math.nan
    lengths = [0, 77]
    kd, vd = _dirty(k, v, lengths)
    out = oc.tree_attention(q, kd, vd, dk, dv, mask.cuda(), lengths=torch.tensor(lengths))
    vis = torch.cat([(torch.arange(S)[None] < torch.tensor(lengths)[:, None])[:, None].expand(B, T, S), mask], 2)
    want, _, tol, _ = R.attend(q, torch.cat([kd, dk], 1), torch.cat([vd, dv], 1), vis.cuda())
    R.check(out, want, tol)
    assert not out[0, -2:].any()


def test_tree_over_a_cache_of_no_capacity():
    import orthocache_b200 as oc
    g = _gen(3)
    q, k, v = _qkv(g, 1, 6, 4, 2, 0, 128, BF)
    dk, dv = _randn(g, 1, 6, 2, 128), _randn(g, 1, 6, 2, 128)
    mask = R.random_tree(6, g)
    out = oc.tree_attention(q, k, v, dk, dv, mask.cuda())
    want, _, tol, _ = R.attend(q, dk, dv, mask[None].cuda())
    R.check(out, want, tol)


def test_one_node_tree_equals_the_chunk_form():
    """A tree of one node over n tokens is a chunk of one query over n + 1."""
    import orthocache_b200 as oc
    g = _gen(4)
    q, k, v = _qkv(g, 2, 1, 16, 4, 901, 128, BF)
    a = oc.tree_attention(q, k[:, :900], v[:, :900], k[:, 900:], v[:, 900:], torch.ones(1, 1, dtype=torch.bool))
    b = oc.chunk_attention(q, k, v)
    want, _, tol, _ = R.attend(q, k, v, torch.ones(2, 1, 901, dtype=torch.bool).cuda())
    R.check(a, want, tol)
    R.check(b, want, tol)


# ---------------------------------------------------------------------------
# chunk
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,N,Hq,Hkv,S,D,kw", [
    (1, 1, 1, 1, 1, 64, {}),
    (1, 1, 32, 8, 1000, 128, dict(cap=30.0)),
    (2, 1, 16, 2, 300, 256, dict(slopes=True)),
    (2, 3, 6, 2, 65, 64, {}),
    (2, 70, 8, 2, 70, 128, dict(causal=False)),
    (1, 129, 4, 4, 129, 128, {}),
    (2, 200, 8, 2, 777, 128, dict(cap=50.0)),
    (2, 257, 6, 2, 300, 128, dict(prefix=[90, 0])),
    (1, 300, 5, 1, 300, 64, dict(slopes=True)),
    (2, 333, 8, 4, 640, 128, dict(documents=48)),
    (2, 150, 3, 1, 513, 256, dict(documents=100, prefix=[200, 600], slopes=True, cap=15.0)),
    (1, 640, 8, 8, 640, 128, dict(documents=128, slopes=True)),
    (2, 513, 12, 4, 1025, 128, dict(prefix=[1000, 2000], cap=20.0)),
])
def test_chunk_against_float64(B, N, Hq, Hkv, S, D, kw, dtype):
    import orthocache_b200 as oc
    kw = dict(kw)
    g = _gen(B * 100 + N + S)
    q, k, v = _qkv(g, B, N, Hq, Hkv, S, D, dtype)
    lengths = [max(1, S - 61 * b) for b in range(B)]
    k, v = _dirty(k, v, lengths)
    docs = bias = slopes = None
    if "documents" in kw:
        step = kw.pop("documents")
        docs = (torch.arange(S) // step).repeat(B, 1).to(torch.int32)
        docs[:, ::step] = torch.arange(len(range(0, S, step)), dtype=torch.int32) // 2  # ids that come back
        docs[:, S // 3:S // 3 + 7] = -1  # padding in the middle
        for b in range(B):
            k[b, docs[b] < 0] = math.nan
            v[b, docs[b] < 0] = math.nan
    if kw.pop("slopes", False):
        slopes = 2.0 ** (-8.0 * (torch.arange(Hq) + 1) / Hq)
        bias = R.distance_bias(lengths, N, S, slopes).cuda()
    out = oc.chunk_attention(q, k, v, torch.tensor(lengths), documents=docs,
                             slopes=slopes, **{x: (torch.tensor(y) if x == "prefix" else y) for x, y in kw.items()})
    vis = R.chunk_visible(lengths, N, S, kw.get("causal", True), kw.get("prefix"), docs).cuda()
    want, _, tol, _ = R.attend(q, k, v, vis, cap=kw.get("cap", 0.0), bias=bias)
    assert out.dtype == dtype
    R.check(out, want, tol)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N", [5, 300])
def test_rows_without_keys_are_zero(N, dtype):
    """Sequences shorter than the chunk (a batch padded on the left), of one
    token and of none, lengths outside the capacity."""
    import orthocache_b200 as oc
    g = _gen(N)
    B, Hq, Hkv, S, D = 6, 4, 2, 320, 128
    q, k, v = _qkv(g, B, N, Hq, Hkv, S, D, dtype)
    lengths = [N, N - 3, 1, 0, -7, 5000]
    real = [min(max(n, 0), S) for n in lengths]
    kd, vd = _dirty(k, v, real)
    out = oc.chunk_attention(q, kd, vd, torch.tensor(lengths))
    vis = R.chunk_visible(real, N, S).cuda()
    want, _, tol, _ = R.attend(q, kd, vd, vis)
    R.check(out, want, tol)
    assert not out[3].any() and not out[4].any() and not out[1, :3].any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scale_and_zero_queries(dtype):
    import orthocache_b200 as oc
    g = _gen(8)
    q, k, v = _qkv(g, 1, 130, 4, 2, 200, 128, dtype)
    vis = R.chunk_visible([200], 130, 200).cuda()
    for scale in (0.0, 0.02, -0.05):
        out = oc.chunk_attention(q, k, v, scale=scale)
        want, _, tol, _ = R.attend(q, k, v, vis, scale=scale)
        R.check(out, want, tol, f"scale {scale}")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N", [2, 200])
def test_large_scores(N, dtype):
    """Scores up to several hundred: the softmax is nearly one key, and the
    capped form flattens it."""
    import orthocache_b200 as oc
    g = _gen(9)
    q, k, v = _qkv(g, 1, N, 4, 2, 400, 128, dtype)
    q, k = q * 8, k * 8
    vis = R.chunk_visible([400], N, 400).cuda()
    for cap in (0.0, 10.0, 50.0):
        out = oc.chunk_attention(q, k, v, cap=cap)
        want, _, tol, _ = R.attend(q, k, v, vis, cap=cap)
        R.check(out, want, tol, f"cap {cap}")


def test_nonfinite_inputs_stay_in_their_rows():
    """An infinite or NaN query spoils its own row only; a NaN key that a row
    sees makes that row NaN."""
    import orthocache_b200 as oc
    g = _gen(10)
    for dtype, N in ((BF, 3), (BF, 260), (F32, 40)):
        q, k, v = _qkv(g, 1, N, 4, 2, 300, 128, dtype)
        q[0, 1, 2, 5] = math.nan
        out = oc.chunk_attention(q, k, v)
        bad = torch.zeros(1, N, 4, dtype=torch.bool)
        bad[0, 1, 2] = True
        assert torch.equal(out.isnan().all(-1).cpu(), bad) and torch.equal(out.isnan().any(-1).cpu(), bad)


def test_strided_inputs_and_unbatched_shapes():
    import orthocache_b200 as oc
    g = _gen(11)
    B, N, Hq, Hkv, S, D = 2, 40, 8, 2, 150, 128
    q, k, v = _qkv(g, B, N, Hq, Hkv, S, D, BF)
    want = oc.chunk_attention(q, k, v, cap=9.0)
    qt = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    kv = torch.stack([k, v], 2)  # interleaved
    kt = k.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(oc.chunk_attention(qt, kt, kv[:, :, 1], cap=9.0), want)
    odd = torch.empty(B * S * Hkv * D + 1, dtype=BF, device="cuda")[1:].view(B, S, Hkv, D)  # 2-byte aligned
    odd.copy_(k)
    with pytest.raises(oc._lib.OrthoCacheError, match="aligned"):
        oc.chunk_attention(q, odd, v)
    for b in range(B):
        assert torch.equal(oc.chunk_attention(q[b], k[b], v[b], cap=9.0), want[b])
    docs = (torch.arange(S) // 40).to(torch.int32)
    assert torch.equal(oc.chunk_attention(q[0], k[0], v[0], documents=docs),
                       oc.chunk_attention(q[:1], k[:1], v[:1], documents=docs[None])[0])


def test_other_stream_and_graph_replay():
    """On a stream of the user's own, and two captured graphs replayed in turn
    with new inputs: what a graph uses belongs to it."""
    import orthocache_b200 as oc
    g = _gen(12)
    B, Hq, Hkv, S, D = 2, 16, 4, 4000, 128
    q1, k, v = _qkv(g, B, 1, Hq, Hkv, S, D, BF)
    q2 = _randn(g, B, 150, Hq, D)
    lens = torch.tensor([4000, 3100], dtype=torch.int32, device="cuda")
    w = torch.zeros(B, Hkv, S, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for _ in range(2):
            oc.accumulate_attention(q1, k, v, w, lens)
            oc.chunk_attention(q2, k, v, lens, cap=30.0)
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1, w1 = oc.accumulate_attention(q1, k, v, w, lens)
    with torch.cuda.graph(g2):
        o2 = oc.chunk_attention(q2, k, v, lens, cap=30.0)
    for seed in (1, 2):
        h = _gen(seed)
        q1.copy_(_randn(h, B, 1, Hq, D))
        q2.copy_(_randn(h, B, 150, Hq, D))
        lens.copy_(torch.tensor([4000 - 500 * seed, 3100 + 100 * seed]))
        g1.replay()
        g2.replay()
        g1.replay()
        want1, wantw = oc.accumulate_attention(q1, k, v, w, lens)
        assert torch.equal(o1, want1) and torch.equal(w1, wantw)
        assert torch.equal(o2, oc.chunk_attention(q2, k, v, lens, cap=30.0))


# ---------------------------------------------------------------------------
# accumulate
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,N,Hq,Hkv,S,D,cap", [
    (1, 1, 1, 1, 1, 64, 0.0),
    (2, 1, 32, 8, 1500, 128, 0.0),
    (1, 3, 12, 4, 300, 64, 0.0),
    (2, 16, 8, 2, 515, 128, 30.0),
    (3, 40, 8, 2, 200, 128, 0.0),
    (2, 200, 6, 2, 333, 128, 0.0),
    (1, 130, 4, 2, 300, 256, 12.0),
    (2, 300, 8, 4, 900, 64, 0.0),
    (2, 400, 8, 2, 400, 128, 50.0),
])
def test_accumulate_against_float64(B, N, Hq, Hkv, S, D, cap, dtype):
    import orthocache_b200 as oc
    g = _gen(B * 77 + N + S)
    q, k, v = _qkv(g, B, N, Hq, Hkv, S, D, dtype)
    lengths = [max(1, S - 71 * b) for b in range(B)]
    kd, vd = _dirty(k, v, lengths)
    w = torch.rand(B, Hkv, S, generator=g).cuda()
    out, new = oc.accumulate_attention(q, kd, vd, w, torch.tensor(lengths), cap=cap)
    vis = R.chunk_visible(lengths, N, S).cuda()
    want, p, tol, rel = R.attend(q, kd, vd, vis, cap=cap)
    R.check(out, want, tol, "out")
    sums, stol = R.column_sums(p, rel, Hkv)
    R.check(new, w.double() + sums, stol + 2.0 ** -24 * (w.double() + sums), "weights")
    for b, n in enumerate(lengths):
        assert torch.equal(new[b, :, n:], w[b, :, n:])
    # from nothing, and in place
    out0, w0 = oc.accumulate_attention(q, kd, vd, None, torch.tensor(lengths), cap=cap)
    R.check(w0, sums, stol, "weights from zero")
    assert torch.equal(out0, out)
    kept = w.clone()
    _, same = oc.accumulate_attention(q, kd, vd, kept, torch.tensor(lengths), cap=cap, out_weights=kept)
    assert same is kept and torch.equal(kept, new)


@pytest.mark.parametrize("N", [1, 300])
def test_accumulate_is_repeatable_and_ignores_empty_rows(N):
    import orthocache_b200 as oc
    g = _gen(N)
    B, Hq, Hkv, S, D = 3, 8, 2, 350, 128
    q, k, v = _qkv(g, B, N, Hq, Hkv, S, D, BF)
    lengths = [350, 4, 0]
    kd, vd = _dirty(k, v, lengths)
    runs = [oc.accumulate_attention(q, kd, vd, None, torch.tensor(lengths)) for _ in range(3)]
    for out, w in runs[1:]:
        assert torch.equal(out, runs[0][0]) and torch.equal(w, runs[0][1])
    _, p, _, rel = R.attend(q, kd, vd, R.chunk_visible(lengths, N, S).cuda())
    sums, tol = R.column_sums(p, rel, Hkv)
    R.check(runs[0][1], sums, tol)
    assert not runs[0][1][2].any()


# ---------------------------------------------------------------------------
# far offsets, and the operators in a row
# ---------------------------------------------------------------------------
def test_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements, the attended tokens at its end."""
    import orthocache_b200 as oc
    B, S, Hkv, D, N = 2, 1 << 20, 8, 192 - 64, 3
    k = torch.zeros((B, S, Hkv, D), dtype=BF, device="cuda")
    v = torch.zeros_like(k)
    assert k.numel() >= 1 << 31
    g = _gen(21)
    tail = 700
    kt, vt = _randn(g, B, tail, Hkv, D), _randn(g, B, tail, Hkv, D)
    k[:, S - tail:] = kt
    v[:, S - tail:] = vt
    q = _randn(g, B, N, 16, D)
    docs = torch.full((B, S), 1, dtype=torch.int32, device="cuda")
    docs[:, :S - tail] = 2
    out = oc.chunk_attention(q, k, v, documents=docs)
    want, _, tol, _ = R.attend(q, kt, vt, R.chunk_visible([tail] * B, N, tail).cuda())
    R.check(out, want, tol)
    w = torch.zeros(B, Hkv, S, device="cuda")
    w[:, :, S - tail:] = 1.0
    ke, ve, _, index, left = oc.evict_tokens(k, v, w, tail)
    assert torch.equal(ke, kt) and torch.equal(ve, vt) and left.tolist() == [tail] * B
    assert torch.equal(index[1, 3].cpu(), torch.arange(S - tail, S, dtype=torch.int32))


@pytest.mark.parametrize("dtype,D", [(BF, 128), (BF, 64), (F32, 64)])
def test_prompt_evict_verify(dtype, D):
    """As a serving loop runs them: a prompt chunk whose weights start the sums,
    some decoded tokens that add to them, the cut, and a drafted tree over
    what is left."""
    import orthocache_b200 as oc
    g = _gen(31)
    B, Hq, Hkv, S, keep, recent, T = 2, 8, 2, 420, 100, 20, 12
    q, k, v = _qkv(g, B, 300, Hq, Hkv, S, D, dtype)
    lens = torch.tensor([300, 260], dtype=torch.int32, device="cuda")
    out, w = oc.accumulate_attention(q, k, v, None, lens)
    for _ in range(3):
        lens += 1
        out, _ = oc.accumulate_attention(_randn(g, B, 1, Hq, D, dtype=dtype), k, v, w, lens, out_weights=w)
    total = w.sum(-1).cpu()
    # each row's weights sum to 1: the rows of 300 queries (260 of them real in row 1) and three steps
    rows = torch.tensor([[303.0 * Hq // Hkv], [263.0 * Hq // Hkv]])
    assert torch.allclose(total, rows.expand(B, Hkv), rtol=1e-4)
    k2, v2, w2, index, left = oc.evict_tokens(k, v, w, keep, recent, lens)
    n = lens.tolist()
    for b in range(B):
        for h in range(Hkv):
            pick = R.evict_index(w[b, h].cpu(), n[b], keep, recent)
            assert index[b, h].tolist() == pick
            assert torch.equal(k2[b, :, h], k[b, pick, h]) and torch.equal(v2[b, :, h], v[b, pick, h])
    assert left.tolist() == [keep, keep]
    qt = _randn(g, B, T, Hq, D, dtype=dtype)
    dk, dv = _randn(g, B, T, Hkv, D, dtype=dtype), _randn(g, B, T, Hkv, D, dtype=dtype)
    mask = R.random_tree(T, g)
    got = oc.tree_attention(qt, k2, v2, dk, dv, mask, left)
    vis = torch.cat([torch.ones(B, T, keep, dtype=torch.bool), mask.expand(B, T, T)], 2).cuda()
    want, _, tol, _ = R.attend(qt, torch.cat([k2, dk], 1), torch.cat([v2, dv], 1), vis)
    R.check(got, want, tol)


def test_refusals():
    import orthocache_b200 as oc
    g = _gen(41)
    q, k, v = _qkv(g, 2, 4, 8, 2, 64, 128, BF)
    mask = torch.ones(4, 4, dtype=torch.bool)
    dk, dv = k[:, :4], v[:, :4]
    bad = [
        (ValueError, lambda: oc.chunk_attention(q[:, :, :7], k, v)),
        (ValueError, lambda: oc.chunk_attention(q[..., :64], k, v)),
        (ValueError, lambda: oc.chunk_attention(q[:, :0], k, v)),
        (ValueError, lambda: oc.chunk_attention(q, k, v[:, :60])),
        (ValueError, lambda: oc.chunk_attention(q[..., :96], k[..., :96], v[..., :96])),
        (ValueError, lambda: oc.chunk_attention(q, k, v, torch.tensor([64]))),
        (TypeError, lambda: oc.chunk_attention(q, k, v, torch.tensor([64.0, 3.0]))),
        (ValueError, lambda: oc.chunk_attention(q, k, v, prefix=torch.tensor([1, 2, 3]))),
        (ValueError, lambda: oc.chunk_attention(q, k, v, documents=torch.zeros(2, 63, dtype=torch.int32))),
        (ValueError, lambda: oc.chunk_attention(q, k, v, slopes=torch.ones(2))),
        (ValueError, lambda: oc.chunk_attention(q, k, v, cap=-1.0)),
        (ValueError, lambda: oc.chunk_attention(q, k, v, cap=math.inf)),
        (ValueError, lambda: oc.chunk_attention(q, k, v, scale=math.nan)),
        (ValueError, lambda: oc.tree_attention(q, k, v, dk, dv[:, :3], mask)),
        (ValueError, lambda: oc.tree_attention(q, k, v, dk, dv, mask[:3])),
        (TypeError, lambda: oc.tree_attention(q, k, v, dk, dv, mask.float())),
        (ValueError, lambda: oc.tree_attention(q, k[:1], v[:1], dk, dv, mask)),
        (ValueError, lambda: oc.tree_attention(q, k[0], v[0], dk, dv, mask, block_table=torch.zeros(2, 1).int())),
        (ValueError, lambda: oc.accumulate_attention(q, k, v, torch.zeros(2, 64, 2).cuda())),
        (ValueError, lambda: oc.accumulate_attention(q, k, v, out_weights=torch.zeros(2, 2, 64))),
        (ValueError, lambda: oc.accumulate_attention(q, k, v, out_weights=torch.zeros(2, 64, 2).cuda().transpose(1, 2))),
        (ValueError, lambda: oc.evict_tokens(k, v, torch.zeros(2, 2, 64).cuda(), 0)),
        (ValueError, lambda: oc.evict_tokens(k, v, torch.zeros(2, 2, 64).cuda(), 65)),
        (ValueError, lambda: oc.evict_tokens(k, v, torch.zeros(2, 2, 64).cuda(), 8, 9)),
        (ValueError, lambda: oc.evict_tokens(k, v, torch.zeros(2, 64, 2).cuda(), 8)),
    ]
    for i, (exc, call) in enumerate(bad):
        with pytest.raises(exc):
            call()
            pytest.fail(f"call {i} was not refused")
    wide = torch.ones(257, 257, dtype=torch.bool)
    x = _randn(g, 1, 257, 2, 128)
    with pytest.raises(oc._lib.OrthoCacheError, match="256"):
        oc.tree_attention(x, k[:1], v[:1], x, x, wide)


# ---------------------------------------------------------------------------
# the cut of the keys over CTAs, and the softmax's reference point
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,D,Hq,Hkv", [(BF, 128, 8, 2), (BF, 128, 3, 3), (BF, 64, 16, 1), (BF, 256, 4, 2),
                                            (F32, 64, 6, 2)])
@pytest.mark.parametrize("T", [1, 11, 70])
def test_ragged_batch_cut_over_many_ctas(T, D, Hq, Hkv, dtype):
    """Sequences of very different lengths (none, one token, thousands), whose
    key tiles are dealt out over all CTAs; every batch row, head and node."""
    import orthocache_b200 as oc
    g = _gen(T + D)
    lengths = [7000, 1, 0, 2500, 129, 64]
    B, S = len(lengths), 7040
    q, k, v = _qkv(g, B, T, Hq, Hkv, S, D, dtype)
    dk, dv = _randn(g, B, T, Hkv, D, dtype=dtype), _randn(g, B, T, Hkv, D, dtype=dtype)
    mask = R.random_tree(T, g)
    kd, vd = _dirty(k, v, lengths)
    lens = torch.tensor(lengths)
    out = oc.tree_attention(q, kd, vd, dk, dv, mask, lens)
    vis = torch.cat([(torch.arange(S)[None] < lens[:, None])[:, None].expand(B, T, S), mask.expand(B, T, T)], 2).cuda()
    want, _, tol, _ = R.attend(q, torch.cat([kd, dk], 1), torch.cat([vd, dv], 1), vis)
    R.check(out, want, tol, "tree")
    out, w = oc.accumulate_attention(q, kd, vd, None, lens)
    want, p, tol, rel = R.attend(q, kd, vd, R.chunk_visible(lengths, T, S).cuda())
    R.check(out, want, tol, "chunk")
    sums, stol = R.column_sums(p, rel, Hkv)
    R.check(w, sums, stol, "weights")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kw", [{}, dict(cap=100.0), dict(slopes=-0.6), dict(slopes=0.9), dict(slopes=-0.2, cap=20.0),
                                dict(slopes=0.3, prefix=[500]), dict(causal=False, slopes=-0.4)])
@pytest.mark.parametrize("N", [3, 160])
def test_scores_that_grow_away_from_the_query(N, kw, D):
    """The largest scores lie farthest from the query (by the keys, or by a
    negative bias): a softmax that takes its reference point from the nearest
    keys has to move it, by far more than float32 holds."""
    import orthocache_b200 as oc
    kw = dict(kw)
    g = _gen(N + D)
    B, Hq, Hkv, S = 1, 4, 2, 900
    q, k, v = _qkv(g, B, N, Hq, Hkv, S, D, BF)
    # one direction that every query shares; the keys have the more of it the farther back they lie
    q = q * 0.3
    q[..., 0] = 24.0
    k[..., 0] = (torch.linspace(120.0, -120.0, S).view(1, S, 1) * D ** 0.5 / 11.3).to(BF).cuda()
    bias = slopes = None
    if "slopes" in kw:
        slopes = kw.pop("slopes") * torch.linspace(0.5, 1.0, Hq)
        bias = R.distance_bias([S], N, S, slopes).cuda()
    prefix = kw.pop("prefix", None)
    out = oc.chunk_attention(q, k, v, slopes=slopes, prefix=None if prefix is None else torch.tensor(prefix), **kw)
    vis = R.chunk_visible([S], N, S, kw.get("causal", True), prefix).cuda()
    want, _, tol, _ = R.attend(q, k, v, vis, cap=kw.get("cap", 0.0), bias=bias)
    R.check(out, want, tol)


def test_padding_fills_whole_tiles():
    """Documents separated by padding longer than a tile, with queries of the
    padding among the rows of a tile."""
    import orthocache_b200 as oc
    g = _gen(77)
    B, N, Hq, Hkv, S, D = 1, 1200, 2, 2, 1200, 128
    q, k, v = _qkv(g, B, N, Hq, Hkv, S, D, BF)
    docs = torch.full((B, S), -1, dtype=torch.int32)
    docs[:, :200], docs[:, 700:] = 5, 9
    docs[:, 900:1190] = 5
    k[docs.cuda() < 0] = math.nan
    v[docs.cuda() < 0] = math.inf
    out = oc.chunk_attention(q, k, v, documents=docs)
    want, _, tol, _ = R.attend(q, k, v, R.chunk_visible([S], N, S, True, None, docs).cuda())
    R.check(out, want, tol)
    assert not out[:, 200:700].any()


def test_no_wait_gave_up():
    from orthocache_b200 import _lib
    torch.cuda.synchronize()
    assert _lib.load().oc_device_status(0) == 0
