"""Float64 reference of the token-level operators and the error bounds their
kernels are held to.

``attend`` takes the visibility of every (query, key) pair as a bool tensor and
returns the output, the weights p, and per output element the bound

    out_type * |out| + p_type * A + fp32 * A,        A = sum_j p_j |v_j|

with half a step per rounding (``torch.finfo(t).eps / 2``): out_type the
rounding of the output, p_type that of the weights where the kernel multiplies
bfloat16 (numerator only: sum_j p_j (1 + d_j) v_j with |d_j| <= eps / 2), and fp32
the float32 arithmetic: with delta = (D + 16) 2^-24 max_j scale sum_d |q_d k_d|
+ 2^-21 max|s| (the dot product's rounding in any order, and the score's own:
the scale, the cap's tanh, the bias and log2(e) are a few float32 roundings of
values up to |s|), a weight moves by at most a factor exp(2 delta), the sums of n
terms add 2 (n + 16) 2^-24 and the exponential 2^-21.
"""
import math

import torch


def heads(x, G):
    return x.double().repeat_interleave(G, dim=2) if G > 1 else x.double()


def attend(q, k, v, visible, scale=None, cap=0.0, bias=None, exact_p=False):
    """q (B, N, Hq, D), k / v (B, S, Hkv, D), visible (B, N, S) -> out, p (B, Hq, N, S), tol (out's shape)."""
    B, N, Hq, D = q.shape
    S, G = k.shape[1], Hq // k.shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    usable = visible.any(1)[:, :, None, None]  # what nobody sees does not exist
    kk, vv = (torch.where(usable, t, torch.zeros((), dtype=t.dtype, device=t.device)) for t in (k, v))
    kk, vv = heads(kk, G), heads(vv, G)
    s = torch.einsum("bnhd,bshd->bhns", q.double(), kk) * scale
    amax = (torch.einsum("bnhd,bshd->bhns", q.double().abs(), kk.abs()) * abs(scale)).amax(-1) if S else s.new_zeros(
        s.shape[:3])
    if cap > 0:
        s = cap * torch.tanh(s / cap)
    if bias is not None:
        s = s + bias
    big = s.masked_fill(~visible[:, None], 0).abs().amax(-1) if S else amax
    s = s.masked_fill(~visible[:, None], -math.inf)
    m = s.amax(-1, keepdim=True) if S else s.new_zeros(s.shape[:3] + (1,))
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    tot = p.sum(-1, keepdim=True)
    p = p / torch.where(tot == 0, torch.ones_like(tot), tot)
    out = torch.einsum("bhns,bshd->bnhd", p, vv)
    A = torch.einsum("bhns,bshd->bnhd", p, vv.abs())
    # 2^-21 |s|: eight float32 roundings of values no larger than |s|
    delta = (D + 16) * 2.0 ** -24 * amax + 2.0 ** -21 * (big + cap)
    rel = 2 * delta + 2 * (S + 16) * 2.0 ** -24 + 2.0 ** -21  # (B, Hq, N)
    half = torch.finfo(q.dtype).eps / 2
    p_half = 2.0 ** -8 if q.dtype == torch.bfloat16 and not exact_p else 0.0
    # 1.0625: products of two of the terms
    tol = 1.0625 * (half * out.abs() + (p_half + rel.transpose(1, 2)[..., None]) * A) + 1e-30
    return out, p, tol, rel


def column_sums(p, rel, Hkv):
    """Sum of the weights over the query rows of each KV head, with its bound."""
    B, Hq, N, S = p.shape
    w = p.view(B, Hkv, Hq // Hkv, N, S).sum((2, 3))
    tol = (p * (rel[..., None] + (N * Hq // Hkv + 8) * 2.0 ** -24)).view(B, Hkv, Hq // Hkv, N, S).sum((2, 3))
    return w, 1.0625 * tol + 1e-12  # a weight below 2^-126 may be flushed to zero


def check(got, want, tol, what=""):
    assert got.shape == want.shape, (got.shape, want.shape)
    err = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all(), f"{what}: not finite"
    worst = float((err / tol).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: error {float(err.max()):.3e}, {worst:.2f} of the bound"


def chunk_visible(lengths, N, S, causal=True, prefix=None, documents=None):
    """(B, N, S) bool on the CPU, by the definition, pair by pair over rows."""
    B = len(lengths)
    j = torch.arange(S)
    rows = []
    for b in range(B):
        pos = lengths[b] - N + torch.arange(N)
        vis = (j[None] < lengths[b]) & (pos[:, None] >= 0)
        if causal:
            ok = j[None] <= pos[:, None]
            if prefix is not None:
                ok = ok | (j[None] < prefix[b])
            vis = vis & ok
        if documents is not None:
            d = documents[b].cpu().long()
            mine = d[pos.clamp(0, max(S - 1, 0))] if S else torch.zeros(N, dtype=torch.long)
            vis = vis & (mine[:, None] == d[None]) & (mine[:, None] >= 0)
        rows.append(vis)
    return torch.stack(rows)


def distance_bias(lengths, N, S, slopes):
    pos = torch.as_tensor(lengths)[:, None] - N + torch.arange(N)[None]
    far = (pos[:, :, None] - torch.arange(S)).abs().double()
    return -slopes.double().cpu()[None, :, None, None] * far[:, None]


def random_tree(n, gen):
    """Ancestor mask (n, n) of a random tree with a few roots."""
    mask = torch.zeros(n, n, dtype=torch.bool)
    for t in range(n):
        p = int(torch.randint(max(-1, t - 5), t, (1,), generator=gen)) if t else -1
        if p >= 0:
            mask[t] = mask[p]
        mask[t, t] = True
    return mask


def evict_index(w, n, keep, recent):
    """Kept positions of one head (CPU float32 weights w), ascending."""
    if n <= keep:
        return list(range(n))
    key = [(math.inf if math.isnan(x) else x, math.isnan(x)) for x in w[:n - recent].tolist()]
    order = sorted(range(n - recent), key=lambda i: (not key[i][1], -key[i][0], i))
    return sorted(order[:keep - recent]) + list(range(n - recent, n))
