"""Eviction by accumulated weight against a plain selection, bit for bit."""
import math

import pytest
import torch

import token_ref as R

pytestmark = pytest.mark.gpu


def _check(k, v, w, keep, recent, lengths):
    import orthocache_b200 as oc
    B, S, H, D = k.shape
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    k2, v2, w2, index, left = oc.evict_tokens(k, v, w, keep, recent, lens)
    real = [S] * B if lengths is None else [min(max(n, 0), S) for n in lengths]
    assert left.tolist() == [min(n, keep) for n in real] and left.dtype == torch.int32
    wc = w.cpu()
    for b in range(B):
        for h in range(H):
            pick = R.evict_index(wc[b, h], real[b], keep, recent)
            n = len(pick)
            assert index[b, h, :n].tolist() == pick, (b, h)
            assert (index[b, h, n:] == -1).all() and not w2[b, h, n:].any()
            assert torch.equal(k2[b, :n, h], k[b, pick, h]) and torch.equal(v2[b, :n, h], v[b, pick, h])
            assert torch.equal(w2[b, h, :n].cpu().view(torch.int32), wc[b, h, pick].view(torch.int32))
            assert not k2[b, n:, h].any() and not v2[b, n:, h].any()


def _cache(seed, B, S, H, D, dtype):
    g = torch.Generator()
    g.manual_seed(seed)
    k, v = (torch.randn(B, S, H, D, generator=g).to(dtype).cuda() for _ in range(2))
    return g, k, v


@pytest.mark.parametrize("B,S,H,D,keep,recent,lengths,dtype", [
    (1, 1, 1, 64, 1, 0, None, torch.float32),
    (1, 2, 1, 8, 1, 1, None, torch.bfloat16),
    (2, 37, 3, 64, 5, 0, [37, 4], torch.bfloat16),
    (2, 300, 2, 128, 100, 100, [300, 150], torch.bfloat16),
    (3, 1025, 2, 64, 1024, 17, [1025, 1024, 1000], torch.float32),
    (4, 2050, 1, 256, 33, 32, [0, -5, 9999, 34], torch.bfloat16),
    (1, 5000, 8, 128, 1250, 128, [4999], torch.bfloat16),
    (2, 40000, 2, 64, 9999, 77, [40000, 33333], torch.bfloat16),
])
def test_evict(B, S, H, D, keep, recent, lengths, dtype):
    g, k, v = _cache(S + keep, B, S, H, D, dtype)
    w = torch.exp(2 * torch.randn(B, H, S, generator=g) - 2)
    _check(k, v, (w * 64).round().div(64).cuda(), keep, recent, lengths)  # many equal weights
    _check(k, v, w.cuda(), keep, recent, lengths)


def test_equal_negative_infinite_and_nan_weights():
    g, k, v = _cache(3, 1, 3000, 6, 64, torch.bfloat16)
    w = torch.zeros(1, 6, 3000)
    w[0, 1] = torch.randn(3000, generator=g)  # negative ones too
    w[0, 2] = -0.0
    w[0, 2, ::3] = 0.0
    w[0, 3, 100:140] = math.inf
    w[0, 3, 200:260] = -math.inf
    w[0, 4] = torch.randn(3000, generator=g).abs()
    w[0, 4, 5::70] = math.nan
    w[0, 4, 7::70] = math.inf
    w[0, 5] = torch.rand(3000, generator=g) * 1e-40  # subnormal
    _check(k, v, w.cuda(), 50, 10, None)
    _check(k, v, w.cuda(), 2990, 0, None)


def test_evict_in_a_graph_and_unbatched():
    import orthocache_b200 as oc
    g, k, v = _cache(7, 2, 900, 4, 128, torch.bfloat16)
    w = torch.rand(2, 4, 900, generator=g).cuda()
    lens = torch.tensor([900, 500], dtype=torch.int32, device="cuda")
    oc.evict_tokens(k, v, w, 64, 8, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = oc.evict_tokens(k, v, w, 64, 8, lens)
    for seed in range(2):
        w.copy_(torch.rand(2, 4, 900, generator=g))
        lens.copy_(torch.tensor([30 + 400 * seed, 900 - 300 * seed]))
        graph.replay()
        for a, b in zip(got, oc.evict_tokens(k, v, w, 64, 8, lens)):
            assert torch.equal(a, b)
    one = oc.evict_tokens(k[0], v[0], w[0], 64, 8)
    all_ = oc.evict_tokens(k, v, w, 64, 8)
    for a, b in zip(one[:4], all_[:4]):
        assert torch.equal(a, b[0])
