"""The accumulating attention on both sides of the limit of its stored scores,
and where it multiplies again for a negative scale.  Bounds: ``token_ref``."""
import pytest
import torch

import token_ref as R

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _randn(g, *shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("S,Hkv", [(32768, 16), (32800, 16), (60000, 16), (140000, 32)])
def test_both_sides_of_the_limit(S, Hkv, dtype):
    """One pass, groups of 4, of 4 and of 2 batch rows, and rows that are beyond the limit by themselves."""
    import orthocache_b200 as oc
    g = torch.Generator("cuda").manual_seed(S)
    B, N, G, D = 8, 8, 4, 64
    q = _randn(g, B, N, G * Hkv, D, dtype=dtype)
    k, v = _randn(g, B, S, Hkv, D, dtype=dtype), _randn(g, B, S, Hkv, D, dtype=dtype)
    lengths = [S, S - 1, S - 33, 20000, 5, 64, 1, 0]
    if Hkv == 32:
        B, lengths = 2, [S, 100000]
        q, k, v = q[:2], k[:2], v[:2]
    before = torch.rand(B, Hkv, S, generator=g, device="cuda")
    out, sums = oc.accumulate_attention(q, k, v, None, torch.tensor(lengths))
    out2, added = oc.accumulate_attention(q, k, v, before, torch.tensor(lengths))
    assert torch.equal(out2, out) and torch.equal(added, before + sums)
    rows = torch.tensor([float(min(n, N) * G) for n in lengths], device="cuda")  # each row's weights sum to 1
    assert ((sums.double().sum(-1) - rows[:, None]).abs() <= 1e-4 * rows[:, None]).all()
    for b, h in ((0, 0), (1, 15), (2, 7), (3, 3), (4, 9), (6, 1), (7, 0))[:2 if B == 2 else 7]:
        heads = slice(h * G, (h + 1) * G)
        want, p, tol, rel = R.attend(q[b:b + 1, :, heads], k[b:b + 1, :, h:h + 1], v[b:b + 1, :, h:h + 1],
                                     R.chunk_visible(lengths[b:b + 1], N, S).cuda())
        R.check(out[b:b + 1, :, heads], want, tol, "out")
        ws, wtol = R.column_sums(p, rel, 1)
        R.check(sums[b:b + 1, h:h + 1], ws, wtol, "sums")


@pytest.mark.parametrize("N,G", [(17, 1), (8, 3), (4, 8)])
@pytest.mark.parametrize("scale", [-0.05, 0.0])
@pytest.mark.parametrize("cap", [0.0, 9.0])
def test_scales_of_either_sign_at_256_channels(N, G, scale, cap):
    import orthocache_b200 as oc
    g = torch.Generator("cuda").manual_seed(N)
    B, Hkv, S, D = 2, 2, 700, 256
    q = _randn(g, B, N, G * Hkv, D, dtype=BF)
    k, v = _randn(g, B, S, Hkv, D, dtype=BF), _randn(g, B, S, Hkv, D, dtype=BF)
    lengths = [S, 133]
    out, sums = oc.accumulate_attention(q, k, v, None, torch.tensor(lengths), scale=scale, cap=cap)
    want, p, tol, rel = R.attend(q, k, v, R.chunk_visible(lengths, N, S).cuda(), scale=scale, cap=cap)
    R.check(out, want, tol, "out")
    ws, wtol = R.column_sums(p, rel, Hkv)
    R.check(sums, ws, wtol, "sums")
