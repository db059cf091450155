"""Lengths and prefixes as numbers: Python and NumPy integers, tensors without
a dimension, and what an unbatched call hands on to the next."""
import numpy as np
import pytest
import torch

import token_ref as R

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _inputs(N=5, S=300, Hq=4, Hkv=2, D=64, dtype=F32):
    g = torch.Generator()
    g.manual_seed(N + S)
    return [torch.randn(*s, generator=g).to(dtype).cuda() for s in ((N, Hq, D), (S, Hkv, D), (S, Hkv, D))]


@pytest.mark.parametrize("dtype", [F32, BF])
def test_an_unbatched_loop_hands_its_length_on(dtype):
    """Prompt, cut, drafted tokens and a chunk without the batch dimension: the length that the cut returns is the
    length that the next calls take."""
    import orthocache_b200 as oc
    q, k, v = _inputs(dtype=dtype)
    n = torch.tensor(280, device="cuda")
    out, w = oc.accumulate_attention(q, k, v, None, n)
    out_b, w_b = oc.accumulate_attention(q[None], k[None], v[None], None, torch.tensor([280]))
    assert torch.equal(out, out_b[0]) and torch.equal(w, w_b[0])
    k2, v2, w2, index, left = oc.evict_tokens(k, v, w, 90, 20, n)
    for a, b in zip((k2, v2, w2, index, left), oc.evict_tokens(k[None], v[None], w[None], 90, 20, torch.tensor([280]))):
        assert torch.equal(a, b[0])
    assert left.shape == () and int(left) == 90
    dk, dv, mask = k[:5].contiguous(), v[:5].contiguous(), R.random_tree(5, torch.Generator().manual_seed(1))
    got = oc.tree_attention(q, k2, v2, dk, dv, mask, left)
    want = oc.tree_attention(q[None], k2[None], v2[None], dk[None], dv[None], mask, left[None])
    assert torch.equal(got, want[0])
    assert torch.equal(oc.chunk_attention(q, k2, v2, left), oc.chunk_attention(q, k2, v2, 90))
    k3, _, _, _, left3 = oc.evict_tokens(k2, v2, w2, 40, 0, left)
    assert int(left3) == 40 and k3.shape[0] == 40


@pytest.mark.parametrize("number", [np.int64(170), np.int32(170), np.uint8(170), np.array(170), torch.tensor(170),
                                    torch.tensor(170, dtype=torch.int32, device="cpu"), 170])
def test_numbers(number):
    import orthocache_b200 as oc
    q, k, v = _inputs()
    want = oc.chunk_attention(q, k, v, torch.tensor([170]), prefix=torch.tensor([170]))
    assert torch.equal(oc.chunk_attention(q, k, v, number, prefix=number), want)
    two = [x[None].repeat(2, 1, 1, 1) for x in (q, k, v)]
    assert torch.equal(oc.chunk_attention(*two, number), oc.chunk_attention(*two, torch.tensor([170, 170])))


@pytest.mark.parametrize("n,real", [(2 ** 40, 300), (-2 ** 40, 0), (torch.tensor(2 ** 40), 300)])
def test_numbers_beyond_the_range(n, real):
    """As for tensors: the nearest end of the range."""
    import orthocache_b200 as oc
    q, k, v = _inputs()
    assert torch.equal(oc.chunk_attention(q, k, v, n), oc.chunk_attention(q, k, v, torch.tensor([real])))


def test_refused():
    import orthocache_b200 as oc
    q, k, v = _inputs()
    for bad in (torch.tensor(2.0), np.float32(3), torch.tensor(True)):
        with pytest.raises(TypeError):
            oc.chunk_attention(q, k, v, bad)
    with pytest.raises(ValueError, match="documents"):
        oc.chunk_attention(q, k, v, documents=torch.tensor(3))
    mask = torch.ones(5, 5, dtype=torch.bool)
    pool_k, pool_v = torch.zeros(512, 2, 64, device="cuda"), torch.zeros(512, 2, 64, device="cuda")
    for table in (torch.tensor(0), torch.zeros(1, 1, 1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="block_table"):
            oc.tree_attention(q, pool_k, pool_v, k[:5], v[:5], mask, 5, block_table=table)
