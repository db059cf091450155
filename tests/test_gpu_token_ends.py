"""Blocks that end early: units without keys among units with many, whose blocks
leave while their neighbours' copies are under way; every result is right and
no bounded wait gave up.  Bounds: ``token_ref``."""
import pytest
import torch

import token_ref as R

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("N", [40, 130])
def test_empty_units_among_full_ones(N, D, dtype):
    """More units than the even cut takes, most of them of sequences without tokens or of padding alone."""
    import orthocache_b200 as oc
    from orthocache_b200 import _lib
    g = torch.Generator("cuda").manual_seed(N + D)
    B, Hq, Hkv, S = 290, 4, 2, 260
    q, k, v = (torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((B, N, Hq, D), (B, S, Hkv, D), (B, S, Hkv, D)))
    lengths = [S - b % 7 if b % 3 == 0 else 0 for b in range(B)]
    docs = torch.zeros(B, S, dtype=torch.int32)
    docs[::6] = -1
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for documents in (None, docs):
        vis = R.chunk_visible(lengths, N, S, documents=documents)
        for _ in range(3):
            out = oc.chunk_attention(q, k, v, lens, documents=documents)
        empty = ~vis.any(2)
        assert not out[empty.cuda()].any()
        for b in (0, 3, 6, 144, 288):
            want, _, tol, _ = R.attend(q[b:b + 1], k[b:b + 1], v[b:b + 1], vis[b:b + 1].cuda())
            R.check(out[b:b + 1], want, tol)
    torch.cuda.synchronize()
    assert _lib.load().oc_device_status(0) == 0
