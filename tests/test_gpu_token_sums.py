"""Sums of the attention weights for few query rows per KV head, at lengths that
end anywhere inside a tile and sequences shorter than the chunk, through the C
interface with a workspace that holds garbage: the sums depend on the inputs
alone.  Bounds: ``token_ref``."""
import math

import pytest
import torch

import token_ref as R

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _accumulate(q, k, v, lens, garbage):
    """Output and sums of the C entry point, its workspace and results filled with ``garbage``."""
    from orthocache_b200 import _lib
    B, N, Hq, D = q.shape
    S, Hkv = k.shape[1:3]
    code = _lib.dtype_code(k)
    n = _lib.query("oc_token_attention_workspace_bytes", code, B, N, Hq, Hkv, D, S, 1)
    ws = torch.full(((n + 3) // 4,), garbage, device="cuda")
    out, sums = torch.full_like(q, garbage), torch.full((B, Hkv, S), garbage, device="cuda")
    _lib.call("oc_accumulate_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), code, lens.data_ptr(), None,
              sums.data_ptr(), B, N, Hq, Hkv, D, S, 0.0, D ** -0.5, out.data_ptr(), code, ws.data_ptr(), n,
              _lib.stream_ptr(k.device))
    return out, sums


def _check(N, G, D, Hkv, lengths, S, dtype):
    g = torch.Generator()
    g.manual_seed(N * 1000 + G * 100 + D + S)
    B = len(lengths)

    def randn(*shape):
        return torch.randn(shape, generator=g).to(dtype).cuda()

    q, k, v = randn(B, N, Hkv * G, D), randn(B, S, Hkv, D), randn(B, S, Hkv, D)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    behind = torch.arange(S, device="cuda")[None] >= lens[:, None]
    k[behind], v[behind] = math.nan, math.inf
    out, sums = _accumulate(q, k, v, lens, math.nan)
    want, p, tol, rel = R.attend(q, k, v, R.chunk_visible(lengths, N, S).cuda())
    R.check(out, want, tol, "out")
    ws, wtol = R.column_sums(p, rel, Hkv)
    R.check(sums, ws, wtol, "sums")
    for garbage in (1e30, -math.inf, math.inf):
        again, same = _accumulate(q, k, v, lens, garbage)
        assert torch.equal(again, out) and torch.equal(same, sums), garbage


FEW = [(32, 1), (17, 1), (16, 2), (8, 4), (8, 3), (6, 4), (5, 4), (4, 8), (3, 8), (1, 32), (1, 20), (12, 1), (33, 1)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("N,G", FEW)
def test_sums_at_every_length(N, G, D, dtype):
    """Every length from none to two tiles and two: every residue, and chunks longer than their sequence."""
    _check(N, G, D, 2, list(range(131)), 130 + 5, dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("N,G", FEW)
def test_sums_at_every_length_cut_over_many_ctas(N, G, D, dtype):
    """Few units with many tiles, whose runs end inside them; lengths of every residue."""
    lengths = list(range(1500, 1564))
    _check(N, G, D, 1, lengths, 1570, dtype)
