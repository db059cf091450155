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
