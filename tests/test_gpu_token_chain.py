"""A token-level call whose output is, without anything between, the queries of
the block decode layer, whose kernel may start before the one ahead of it on
the stream has ended.  The layer joins its partials in the order they come, so its
results are held to the float64 bound for their own queries, which those of the
call before are far outside.  Bounds: ``token_ref``."""
import ctypes

import pytest
import torch

import token_ref as R

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
HQ, HKV, D = 32, 8, 128


def _decode(lib, q, k, v, ws, outs):
    keep, perm, count, out = outs
    rc = lib.oc_decode_step(q.data_ptr(), k.data_ptr(), v.data_ptr(), 1, 1, 1, HQ, HKV, D, k.shape[0],
                            ctypes.c_float(-float("inf")), ctypes.c_float(5.0), keep.data_ptr(), perm.data_ptr(),
                            count.data_ptr(), out.data_ptr(), 1, ws.data_ptr(), ws.numel(),
                            torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return out.clone()


@pytest.mark.parametrize("S,tokens", [(100, 100), (60, 33), (5000, 4900)])
def test_output_as_queries(S, tokens):
    from orthocache_b200 import _lib
    lib = _lib.load()
    g = torch.Generator("cuda").manual_seed(S)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(BF)

    nb = 16
    keys, values = randn(nb * 512, HKV, D), randn(nb * 512, HKV, D)
    k, v = randn(1, S, HKV, D), 8 * randn(1, S, HKV, D)
    lens = torch.tensor([tokens], dtype=torch.int32, device="cuda")
    queries = [4 * randn(1, 1, HQ, D) for _ in range(12)]
    buf = torch.empty(1, 1, HQ, D, dtype=BF, device="cuda")
    tok_n = lib.oc_token_attention_workspace_bytes(1, 1, 1, HQ, HKV, D, S, 0)
    tok_ws = torch.empty(max(tok_n, 1), dtype=torch.uint8, device="cuda")
    ws = torch.zeros(lib.oc_decode_step_workspace_bytes(1, 1, HQ, HKV, D, nb * 512), dtype=torch.uint8, device="cuda")
    outs = (torch.empty((nb, HKV), dtype=torch.uint8, device="cuda"), torch.empty((nb,), dtype=torch.int32, device="cuda"),
            torch.empty((1,), dtype=torch.int32, device="cuda"), torch.empty((1, HQ, D), dtype=BF, device="cuda"))

    def run(wait):
        fed, got = [], []
        for q in queries:
            assert lib.oc_chunk_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), 1, lens.data_ptr(), 1, None, None,
                                          None, 1, 1, HQ, HKV, D, S, 0.0, 0.1, buf.data_ptr(), 1, tok_ws.data_ptr(),
                                          tok_n, torch.cuda.current_stream().cuda_stream) == 0
            if wait:
                torch.cuda.synchronize()
                fed.append(buf.clone())
            got.append(_decode(lib, buf, keys, values, ws, outs))
        return fed, got

    fed, _ = run(True)
    seen = torch.ones(1, 1, nb * 512, dtype=torch.bool, device="cuda")
    want = [R.attend(q, keys[None], values[None], seen)[0:3:2] for q in fed]  # with its bound
    for (w, tol), (before, _) in zip(want[1:], want):
        assert ((before - w).abs() > 4 * tol).any()
    for _ in range(5):
        _, got = run(False)
        for o, (w, tol) in zip(got, want):
            R.check(o[None], w, tol)
    assert lib.oc_device_status(0) == 0
