"""Token-level attention over a KV cache.

The block operators of this package attend to whole 512-token blocks without
a mask, like the reference (``src/orthocache/indirect_attention.py:29-170``).
The three operators here attend to single tokens of a cache that holds
``lengths[b]`` of its capacity of tokens:

* ``tree_attention``: drafted tokens arranged in a tree, over a contiguous or
  paged cache (``PagedKVCache.attend_tree``); one decoded token is a tree of
  one node;
* ``chunk_attention``: the last ``Sq`` tokens of every sequence over its cache,
  with a causal, prefix or document mask, scores capped by a tanh and a bias
  that grows with the distance;
* ``accumulate_attention``: causal chunk attention that also adds every key's
  attention weight to a running sum, the input of ``evict_tokens``.

Shapes: q (B, Sq, Hq, D), keys and values (B, S, Hkv, D), float32 or bfloat16,
D in {64, 128, 256}, Hq a multiple of Hkv; without the batch dimension all
per-row arguments lose theirs too (a length is then a number or a tensor without
a dimension; either also stands for a whole batch).  q is brought to the keys'
type and the output has it.  Inputs on the CPU are copied to the GPU.  Nothing
waits for the GPU.
Values inside a sequence are finite and at most 2^50 in magnitude, seen by a row
or not (a hidden one has weight zero, and zero times infinity is NaN); what lies
behind lengths[b], in padding or in drafted tokens that no node sees may be
anything.  With a cap, it is at least scale / 4096.
"""
from __future__ import annotations

import functools
import math
import numbers

import torch

from . import _lib
from .paged import PAGE


def _on(x, device=None, dtype=None):
    """``_lib.as_device``, without its checks for a tensor that is already right (a decode step is a few
    microseconds)."""
    if (isinstance(x, torch.Tensor) and x.is_cuda and (device is None or x.device == device) and
            (x.dtype == dtype if dtype is not None else x.dtype != torch.float64) and x.is_contiguous()):
        return x
    return _lib.as_device(x, device=device, dtype=dtype)


def _call(name, device, *args):
    """A library call with ``device`` current, on its current stream."""
    if device.index == torch.cuda.current_device():
        _lib.call(name, *args, _lib.stream_ptr(device))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _lib.stream_ptr(device))


def _int_rows(x, shape, device, what):
    """An int32 device tensor of ``shape`` (None stays None; a number fills it, a tensor without a dimension a row)."""
    if x is None:
        return None
    if isinstance(x, torch.Tensor) and x.dtype == torch.int32 and x.shape == shape and x.device == device and \
            x.is_contiguous():
        return x
    if isinstance(x, numbers.Integral):
        return torch.full(shape, min(max(int(x), -2 ** 31), 2 ** 31 - 1), dtype=torch.int32, device=device)
    t = _on(x, device)
    if t.dtype.is_floating_point or t.dtype == torch.bool:
        raise TypeError(f"{what} must be integers, got {t.dtype}")
    if t.dim() == 0 and len(shape) == 1:
        t = t.expand(shape)
    if t.shape != shape:
        raise ValueError(f"{what} {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype in (torch.int64, torch.uint32, torch.uint64):  # beyond the range: its nearest end, not another number
        t = t.to(torch.int64).clamp(-2 ** 31, 2 ** 31 - 1)
    return t.to(torch.int32).contiguous()


def _cap_scale(cap, scale, dim):
    cap = float(cap or 0.0)
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not (math.isfinite(cap) and cap >= 0.0):
        raise ValueError(f"cap must be finite and >= 0 (0: none), got {cap}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    if cap and abs(scale) > 4096.0 * min(cap, 4096.0):
        raise ValueError(f"with a cap the scale may be 4096 times the cap, and 2^24, at most, got {scale}, {cap}")
    return cap, scale


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device_index, *sizes):
    with torch.cuda.device(device_index):
        return _lib.query("oc_token_attention_workspace_bytes", *sizes)


def _workspace(device, *sizes):
    """Scratch of one call (what it needs depends on the sizes and the device alone)."""
    n = _workspace_bytes(device.index, *sizes)
    return torch.empty((n,), dtype=torch.uint8, device=device), n


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check_heads(q, kv_heads):
    if kv_heads == 0 or q.shape[2] % kv_heads or q.shape[2] == 0:
        raise ValueError(f"{q.shape[2]} query heads are not a multiple of {kv_heads} KV heads")
    if q.shape[3] not in (64, 128, 256):
        raise ValueError(f"head_dim {q.shape[3]} is not 64, 128 or 256")
    if q.shape[0] == 0 or q.shape[1] == 0:
        raise ValueError(f"empty query {tuple(q.shape)}")


def tree_attention(q, keys, values, draft_keys, draft_values, tree_mask, lengths=None, *, block_table=None, cap=0.0,
                   scale=None):
    """Attention of drafted tokens over a cache and their own ancestors.

    Node i (row i of q (B, T, Hq, D), T <= 256) sees every cache token
    j < lengths[b] (default: all) and the drafted tokens s with tree_mask[b, i, s]
    (bool (T, T) or (B, T, T): its ancestors and, usually, itself).
    draft_keys, draft_values: (B, T, Hkv, D).  With ``block_table`` (B, blocks)
    int32, keys and values are a pool of 512-token pages (pages * 512, Hkv, D)
    and logical block j of row b is page block_table[b, j]; tokens of pages
    outside the pool are seen by nobody.  ``cap`` > 0: scores become
    cap * tanh(score / cap); ``scale`` defaults to 1 / sqrt(D).  A row that
    sees no token is zero.  Returns (B, T, Hq, D) in the cache's type.
    """
    k, v = _cache(keys, values)
    dev, dt = k.device, k.dtype
    qq, dk, dv = _on(q, dev, dt), _on(draft_keys, dev, dt), _on(draft_values, dev, dt)
    batched = qq.dim() == 4
    if not batched:
        qq, dk, dv = qq.unsqueeze(0), dk.unsqueeze(0), dv.unsqueeze(0)
        if block_table is None:
            k, v = k.unsqueeze(0), v.unsqueeze(0)
    kdim = 3 if block_table is not None else 4
    if qq.dim() != 4 or k.dim() != kdim or k.shape != v.shape or dk.dim() != 4 or dk.shape != dv.shape:
        raise ValueError(f"incompatible shapes q {tuple(qq.shape)}, keys {tuple(k.shape)}, values {tuple(v.shape)}, "
                         f"draft {tuple(dk.shape)}, {tuple(dv.shape)}")
    B, T, Hq, D = qq.shape
    Hkv = k.shape[-2]
    _check_heads(qq, Hkv)
    if k.shape[-1] != D or dk.shape != (B, T, Hkv, D):
        raise ValueError(f"incompatible shapes q {tuple(qq.shape)}, keys {tuple(k.shape)}, draft {tuple(dk.shape)}")
    table = None
    if block_table is None:
        if k.shape[0] != B:
            raise ValueError(f"keys {tuple(k.shape)} for {B} batch rows")
        S, pages, stride = k.shape[1], 0, 0
    else:
        if k.shape[0] % PAGE or k.shape[0] == 0:
            raise ValueError(f"a pool of {k.shape[0]} tokens is not a whole number of {PAGE}-token pages")
        table = _on(block_table, device=dev)
        if table.dim() == 1:
            table = table.unsqueeze(0)
        if table.dim() != 2:
            raise ValueError(f"block_table {tuple(table.shape)}, expected ({B}, blocks)")
        table = _int_rows(table, (B, table.shape[-1]), dev, "block_table")
        pages, stride = k.shape[0] // PAGE, table.shape[1]
        S = stride * PAGE
    mask = _on(tree_mask, device=dev)
    mask_batched = mask.dim() == 3
    if mask.shape != ((B, T, T) if mask_batched else (T, T)):
        raise ValueError(f"tree_mask {tuple(mask.shape)}, expected ({T}, {T}) or ({B}, {T}, {T})")
    if mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"tree_mask must be bool, got {mask.dtype}")
    lens = _int_rows(lengths, (B,), dev, "lengths")
    cap, scale = _cap_scale(cap, scale, D)
    code = _lib.dtype_code(k)
    out = torch.empty_like(qq)
    ws, ws_bytes = _workspace(dev, code, B, T, Hq, Hkv, D, S, 0)
    _call("oc_tree_attention", dev, _ptr(qq), _ptr(k), _ptr(v), code, _ptr(table), stride, pages, PAGE, _ptr(lens),
          _ptr(dk), _ptr(dv), _ptr(mask), int(mask_batched), B, T, Hq, Hkv, D, S, cap, scale, _ptr(out), code, _ptr(ws),
          ws_bytes)
    return out if batched else out[0]


def _cache(keys, values):
    k = _on(keys)
    if k.dtype not in (torch.float32, torch.bfloat16):
        k = k.float()
    return k, _on(values, k.device, k.dtype)


def _chunk_inputs(q, keys, values, lengths):
    k, v = _cache(keys, values)
    qq = _on(q, k.device, k.dtype)
    batched = k.dim() == 4
    if not batched:
        qq, k, v = qq.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0)
    if qq.dim() != 4 or k.dim() != 4 or k.shape != v.shape or qq.shape[0] != k.shape[0] or qq.shape[3] != k.shape[3]:
        raise ValueError(f"incompatible shapes q {tuple(qq.shape)}, keys {tuple(k.shape)}, values {tuple(v.shape)}")
    _check_heads(qq, k.shape[2])
    return qq, k, v, batched, _int_rows(lengths, (k.shape[0],), k.device, "lengths")


def chunk_attention(q, keys, values, lengths=None, *, causal=True, prefix=None, documents=None, slopes=None, cap=0.0,
                    scale=None):
    """Attention of the last Sq tokens of every sequence over its cache.

    The cache already holds the chunk: query i of row b sits at position
    pos = lengths[b] - Sq + i (lengths default to the capacity S; a row with
    pos < 0 sees nothing, as in a batch padded on the left) and sees key
    j < lengths[b] iff it is allowed by

    * the causal mask: not ``causal``, or j <= pos, or j < prefix[b]
      (``prefix`` (B,): tokens that every query may see);
    * the document mask: ``documents`` (B, S) int in the range of int32, equal at
      pos and j and not negative (negative: padding, seen by nobody).

    Scores: scale * q.k (1 / sqrt(D) by default), then cap * tanh(score / cap)
    if ``cap`` > 0, then minus slopes[head] * |pos - j| (``slopes`` (Hq,)
    float).  A row that sees no key is zero.  Returns (B, Sq, Hq, D) in the
    cache's type.
    """
    qq, k, v, batched, lens = _chunk_inputs(q, keys, values, lengths)
    B, Sq, Hq, D = qq.shape
    S, Hkv, dev = k.shape[1], k.shape[2], k.device
    cap, scale = _cap_scale(cap, scale, D)
    pre = _int_rows(prefix, (B,), dev, "prefix")
    docs = None
    if documents is not None:
        docs = _on(documents, device=dev)
        docs = _int_rows(docs if batched or docs.dim() != 1 else docs.unsqueeze(0), (B, S), dev, "documents")
    sl = None
    if slopes is not None:
        sl = _on(slopes, device=dev, dtype=torch.float32)
        if sl.shape != (Hq,):
            raise ValueError(f"slopes {tuple(sl.shape)}, expected ({Hq},)")
    code = _lib.dtype_code(k)
    out = torch.empty_like(qq)
    ws, ws_bytes = _workspace(dev, code, B, Sq, Hq, Hkv, D, S, 0)
    _call("oc_chunk_attention", dev, _ptr(qq), _ptr(k), _ptr(v), code, _ptr(lens), int(bool(causal)), _ptr(pre),
          _ptr(docs), _ptr(sl), B, Sq, Hq, Hkv, D, S, cap, scale, _ptr(out), code, _ptr(ws), ws_bytes)
    return out if batched else out[0]


def accumulate_attention(q, keys, values, weights=None, lengths=None, *, cap=0.0, scale=None, out_weights=None):
    """Causal ``chunk_attention`` that also sums every key's attention weight.

    Returns (out, new) with new[b, h, j] = weights[b, h, j] + the softmax
    weights that the query rows of KV head h give key j, summed over the Sq
    queries and the Hq / Hkv heads.  ``weights``: (B, Hkv, S) float32, None for
    zeros; entries behind lengths[b] are copied.  ``out_weights``: a contiguous
    float32 CUDA tensor that receives the sums (``weights`` itself to add in
    place, but no other that shares memory with it); a new one by default.
    """
    qq, k, v, batched, lens = _chunk_inputs(q, keys, values, lengths)
    B, Sq, Hq, D = qq.shape
    S, Hkv, dev = k.shape[1], k.shape[2], k.device
    cap, scale = _cap_scale(cap, scale, D)
    shape = (B, Hkv, S) if batched else (Hkv, S)
    w = None
    if weights is not None:
        w = _on(weights, device=dev, dtype=torch.float32)
        if w.shape != shape:
            raise ValueError(f"weights {tuple(w.shape)}, expected {shape}")
    if out_weights is not None:
        o = out_weights
        if not (isinstance(o, torch.Tensor) and o.device == dev and o.dtype == torch.float32 and o.is_contiguous() and
                o.shape == shape):
            raise ValueError(f"out_weights must be a contiguous float32 tensor {shape} on {dev}")
    code = _lib.dtype_code(k)
    if out_weights is None:
        out_weights = torch.empty(shape, dtype=torch.float32, device=dev)
    out = torch.empty_like(qq)
    ws, ws_bytes = _workspace(dev, code, B, Sq, Hq, Hkv, D, S, 1)
    _call("oc_accumulate_attention", dev, _ptr(qq), _ptr(k), _ptr(v), code, _ptr(lens), _ptr(w), _ptr(out_weights), B, Sq,
          Hq, Hkv, D, S, cap, scale, _ptr(out), code, _ptr(ws), ws_bytes)
    return (out if batched else out[0]), out_weights


def evict_tokens(keys, values, weights, keep, recent=0, lengths=None):
    """Cut a cache down to ``keep`` tokens per KV head.

    keys, values (B, S, Hkv, D), weights (B, Hkv, S) float32 (the sums of
    ``accumulate_attention``).  Of the n = lengths[b] tokens (default S) of
    each head the ``recent`` last stay and, of the others, the keep - recent
    with the largest weights (ties: the lower position; NaN is the largest);
    all stay when n <= keep.  Returns (keys, values, weights, index, lengths) of
    the new cache: (B, keep, Hkv, D) twice, (B, Hkv, keep), the tokens' old
    positions (B, Hkv, keep) int32 in ascending order, and min(n, keep) (B,)
    int32; behind the last kept token zeros and index -1.

    The new cache holds ``keep`` tokens and has no room for another: to go on
    decoding, copy it into one of a larger capacity.  Its tokens are numbered
    anew, so a distance bias (``slopes``) or a document mask over it goes by places
    in the new cache; the old positions are in ``index``, one row per KV head.
    """
    k, v = _cache(keys, values)
    w = _on(weights, device=k.device, dtype=torch.float32)
    batched = k.dim() == 4
    if not batched:
        k, v, w = k.unsqueeze(0), v.unsqueeze(0), w.unsqueeze(0)
    if k.dim() != 4 or k.shape != v.shape or w.shape != (k.shape[0], k.shape[2], k.shape[1]):
        raise ValueError(f"incompatible shapes keys {tuple(k.shape)}, values {tuple(v.shape)}, weights "
                         f"{tuple(w.shape)}")
    B, S, H, D = k.shape
    keep, recent = int(keep), int(recent)
    if not 1 <= keep <= S:
        raise ValueError(f"keep {keep} of {S} tokens")
    if not 0 <= recent <= keep:
        raise ValueError(f"recent {recent}, keep {keep}")
    dev, code = k.device, _lib.dtype_code(k)
    lens = _int_rows(lengths, (B,), dev, "lengths")
    ko = torch.empty((B, keep, H, D), dtype=k.dtype, device=dev)
    vo = torch.empty_like(ko)
    wo = torch.empty((B, H, keep), dtype=torch.float32, device=dev)
    index = torch.empty_like(wo, dtype=torch.int32)
    left = torch.empty((B,), dtype=torch.int32, device=dev)
    _call("oc_evict_tokens", dev, _ptr(k), _ptr(v), code, _ptr(w), _ptr(lens), B, S, H, D, keep, recent, _ptr(ko),
          _ptr(vo), _ptr(wo), _ptr(index), _ptr(left))
    return (ko, vo, wo, index, left) if batched else (ko[0], vo[0], wo[0], index[0], left[0])
