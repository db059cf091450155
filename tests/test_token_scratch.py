"""Scratch of the accumulating attention: stored scores only where a call uses
them, and no more than 512 MiB of them."""
import pytest

BF16, F32 = 1, 0
LIMIT = 512 << 20


def _extra(dtype, batch, q_len, q_heads, kv_heads, dim, seq_len):
    """What the accumulating form needs beyond the plain one, without the softmax denominators."""
    from orthocache_b200 import _lib
    f = _lib.load().oc_token_attention_workspace_bytes
    args = (dtype, batch, q_len, q_heads, kv_heads, dim, seq_len)
    return f(*args, 1) - f(*args, 0) - (batch * q_len * q_heads * 4 + 255) // 256 * 256


def test_dtype_codes():
    from orthocache_b200 import _lib
    assert (_lib.OC_BF16, _lib.OC_F32) == (BF16, F32)


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 64), (F32, 128), (F32, 256)])
@pytest.mark.parametrize("batch,kv_heads,seq_len", [(1, 8, 65536), (8, 16, 32768), (16, 32, 8192)])
def test_stored_up_to_the_limit(dtype, dim, batch, kv_heads, seq_len):
    want = batch * kv_heads * 32 * seq_len * 4
    assert want <= LIMIT
    assert _extra(dtype, batch, 8, 4 * kv_heads, kv_heads, dim, seq_len) == want


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 64), (F32, 128), (F32, 256)])
@pytest.mark.parametrize("batch,kv_heads,seq_len", [(8, 16, 65536), (8, 16, 32769), (9, 16, 60000), (64, 32, 8192),
                                                    (100, 8, 131072), (3, 8, 1 << 19)])
def test_never_more_than_the_limit(dtype, dim, batch, kv_heads, seq_len):
    """A batch with more goes by groups of its rows; beside the scores there are the softmax denominators and two
    partials of 32 rows for each of 512 CTAs at most."""
    from orthocache_b200 import _lib
    n = _lib.load().oc_token_attention_workspace_bytes(dtype, batch, 8, 4 * kv_heads, kv_heads, dim, seq_len, 1)
    rest = batch * kv_heads * 32 * 4 + 2 * 512 * 32 * (dim + 2) * 4 + 5 * 256
    assert LIMIT // 4 < n <= LIMIT + rest


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 64), (F32, 128), (F32, 256)])
def test_one_row_beyond_the_limit_is_multiplied_again(dtype, dim):
    assert _extra(dtype, 2, 8, 32, 8, dim, 1 << 20) == 0


@pytest.mark.parametrize("q_len,group", [(17, 1), (8, 4), (3, 8), (4, 8)])
def test_none_where_no_call_stores_them(q_len, group):
    """bfloat16 at 256 channels: more than 16 rows are multiplied again."""
    assert _extra(BF16, 2, q_len, 4 * group, 4, 256, 20000) == 0
    assert _extra(BF16, 2, 16 // group, 4 * group, 4, 256, 20000) > 0
