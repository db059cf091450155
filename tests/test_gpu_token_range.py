"""Large and small values under weights far from one: scores at either end of a
cap, and scores that grow away from the query, with values whose products with
an ill-chosen softmax reference point leave float32 (values may be as large as 2^50).  Bounds: ``token_ref``."""
import pytest
import torch

import token_ref as R

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _randn(g, *shape, dtype=BF):
    return torch.randn(shape, generator=g).to(dtype).cuda()


def _inputs(N, D, S, dtype):
    g = torch.Generator()
    g.manual_seed(N + D)
    B, Hq, Hkv = 2, 4, 2
    return g, _randn(g, B, N, Hq, D, dtype=dtype), _randn(g, B, S, Hkv, D, dtype=dtype), _randn(g, B, S, Hkv, D, dtype=dtype)


ROWS = [(1, BF), (20, BF), (200, BF), (3, F32), (100, F32)]


@pytest.mark.parametrize("N,dtype", ROWS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cap", [5.0, 40.0, 62.0, 70.0])
@pytest.mark.parametrize("sign,power", [(1.0, 49), (1.0, 0), (-1.0, -70), (-1.0, 49)])
def test_saturated_caps(N, dtype, D, cap, sign, power):
    """Every score at the upper or the lower end of the cap."""
    import orthocache_b200 as oc
    S, lengths = 1500, [1500, 1111]
    g, q, k, v = _inputs(N, D, S, dtype)
    q, k, v = q.abs() * 8, sign * 8 * k.abs(), v * 2.0 ** power
    lens = torch.tensor(lengths)
    out, sums = oc.accumulate_attention(q, k, v, None, lens, cap=cap)
    want, p, tol, rel = R.attend(q, k, v, R.chunk_visible(lengths, N, S).cuda(), cap=cap)
    R.check(out, want, tol, "chunk")
    ws, wtol = R.column_sums(p, rel, k.shape[2])
    R.check(sums, ws, wtol, "sums")
    dk, dv = k[:, :N].contiguous(), v[:, :N].contiguous()
    mask = R.random_tree(N, g)
    out = oc.tree_attention(q, k, v, dk, dv, mask, lens, cap=cap)
    past = (torch.arange(S)[None] < lens[:, None])[:, None].expand(2, N, S)
    vis = torch.cat([past, mask.expand(2, N, N)], 2).cuda()
    want, _, tol, _ = R.attend(q, torch.cat([k, dk], 1), torch.cat([v, dv], 1), vis, cap=cap)
    R.check(out, want, tol, "tree")


@pytest.mark.parametrize("N,dtype", ROWS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rise", [9.0, 38.0, 300.0, -38.0])
@pytest.mark.parametrize("cap", [0.0, 45.0, 1000.0])
def test_large_values_under_rising_scores(N, dtype, D, rise, cap):
    """Scores that change by ``rise`` from the nearest key to the farthest, in steps too
    small for any one tile to stand out."""
    import orthocache_b200 as oc
    S = 2500
    _, q, k, v = _inputs(N, D, S, dtype)
    q, k = q * 0.1, k * 0.1
    q[..., 0] = 8.0
    k[..., 0] = (torch.linspace(rise, 0.0, S).view(1, S, 1) * D ** 0.5 / 8.0).to(dtype).cuda()
    v = v * 2.0 ** 49
    out = oc.chunk_attention(q, k, v, cap=cap)
    want, _, tol, _ = R.attend(q, k, v, R.chunk_visible([S] * 2, N, S).cuda(), cap=cap)
    R.check(out, want, tol)


@pytest.mark.parametrize("N", [40, 200])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_that_see_their_first_key_late(N, D):
    """Capped rows whose nearest tiles hold nothing for them, with every score at the lower end of the cap."""
    import orthocache_b200 as oc
    S, cap = 1400, 60.0
    _, q, k, v = _inputs(N, D, S, BF)
    q, k, v = q.abs() * 8, -8 * k.abs(), v * 2.0 ** -60
    docs = torch.full((2, S), 3, dtype=torch.int32)
    docs[:, 600:] = 4
    docs[:, S - N // 2:] = 3  # half of the rows look back over tiles of another document
    out = oc.chunk_attention(q, k, v, documents=docs, cap=cap)
    want, _, tol, _ = R.attend(q, k, v, R.chunk_visible([S] * 2, N, S, documents=docs).cuda(), cap=cap)
    R.check(out, want, tol)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cap,slopes", [(0.0, 0.0), (60.0, 0.0), (100.0, 0.0), (0.0, -0.02)])
def test_large_values_under_rising_scores_in_whole_units(D, cap, slopes):
    """As above with enough batch rows that one CTA walks all tiles of a row: the weights
    rise by 2^55 between the first tile and the last."""
    import orthocache_b200 as oc
    g = torch.Generator()
    g.manual_seed(D)
    B, N, Hq, Hkv, S, rise = 40, 100, 8, 4, 1500, 38.0
    q, k, v = (_randn(g, B, n, h, D) for n, h in ((N, Hq), (S, Hkv), (S, Hkv)))
    q, k = q * 0.1, k * 0.1
    q[..., 0] = 8.0
    if slopes:
        rise = 8.0
    k[..., 0] = (torch.linspace(rise, 0.0, S).view(1, S, 1) * D ** 0.5 / 8.0).to(BF).cuda()
    v = v * 2.0 ** 49
    sl = torch.full((Hq,), slopes) if slopes else None
    out = oc.chunk_attention(q, k, v, cap=cap, slopes=sl)
    bias = None if sl is None else R.distance_bias([S], N, S, sl).cuda()
    for b in range(0, B, 13):
        want, _, tol, _ = R.attend(q[b:b + 1], k[b:b + 1], v[b:b + 1], R.chunk_visible([S], N, S).cuda(), cap=cap, bias=bias)
        R.check(out[b:b + 1], want, tol)
