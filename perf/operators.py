"""Token-level attention operators over a KV cache: their plain forms, the
calls a user makes of the framework's kernels, and the sizes they are timed at.

Four operators that a serving loop runs one after another on one cache:

* ``tree``: attention of a tree of drafted tokens over a contiguous or paged
  cache (one token is a tree of one node);
* ``chunk``: attention of a query chunk over its cache with the scores capped
  by a tanh or biased by the distance, and a causal, prefix or document mask;
* ``accumulate``: causal attention that also adds every key's attention
  weight to a running sum per (batch row, KV head, token);
* ``evict``: the cache cut down to the most recent tokens and those with the
  largest accumulated weights.

With ``own`` false ``run`` computes them in elementary torch operations in
float32; with ``own`` true it calls the framework.
"""
import math

import numpy as np
import torch

own = False

PAGE = 512  # tokens of one page of the framework's paged cache


def _dt(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _es(case):
    return 2 if case["dtype"] == "bf16" else 4


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------
_TREE = dict(op="tree", batch=1, nodes=1, q_heads=32, kv_heads=8, dim=128, capacity=512, length=512, ragged=0.0,
             paged=False, cap=0.0, dtype="bf16")
_CHUNK = dict(op="chunk", batch=1, q_len=1, q_heads=32, kv_heads=8, dim=128, capacity=512, length=512, ragged=0.0,
              causal=True, prefix=0, document=0, slopes=False, cap=0.0, dtype="bf16")
_ACC = dict(op="accumulate", batch=1, q_len=1, q_heads=32, kv_heads=8, dim=128, capacity=512, length=512, ragged=0.0,
            cap=0.0, dtype="bf16")
_EVICT = dict(op="evict", batch=1, kv_heads=8, dim=128, capacity=512, length=512, ragged=0.0, keep=128, recent=32,
              dtype="bf16")


def listed():
    return [
        # one token on a short cache: what an ordinary decode step costs when latency is all there is
        dict(_TREE, name="tree_one_token", capacity=640, length=601),
        # sixteen drafted tokens verified against the 64K-token cache of the decode benchmark
        dict(_TREE, name="tree_16_on_64k", nodes=16, capacity=65536, length=65500),
        # a batch of paged sequences of different lengths, a wide tree each: the cache's tokens are read once for
        # 61 nodes x 4 heads
        dict(_TREE, name="tree_61_paged", batch=4, nodes=61, capacity=32768, length=32003, ragged=0.6, paged=True,
             cap=30.0),
        # the 256-channel heads of the decode stack's layers, a batch of 8, a few drafted tokens
        dict(_TREE, name="tree_8_dim256", batch=8, nodes=8, q_heads=32, kv_heads=16, dim=256, capacity=8192,
             length=7777, ragged=0.3),
        # chunked prefill: 2048 new tokens behind a 30K-token past, scores capped
        dict(_CHUNK, name="chunk_capped_32k", q_len=2048, capacity=32768, length=32768, cap=50.0),
        # packed documents of about a thousand tokens, distance bias; an odd total length
        dict(_CHUNK, name="chunk_documents", q_len=12001, q_heads=16, kv_heads=8, capacity=12001, length=12001,
             document=1024, slopes=True),
        # float32, prefix mask, padded batch, odd sizes
        dict(_CHUNK, name="chunk_prefix_f32", batch=3, q_len=333, q_heads=12, kv_heads=4, dim=64, capacity=1001,
             length=999, ragged=0.5, prefix=200, dtype="f32"),
        # one decode step of the 64K-token cache that keeps the running weights
        dict(_ACC, name="accumulate_one_64k", capacity=65536, length=65533),
        # a prompt chunk whose weights start the running sum
        dict(_ACC, name="accumulate_chunk", batch=2, q_len=1024, capacity=8192, length=8192, ragged=0.25),
        # a short cache in a batch, cut to a small budget
        dict(_EVICT, name="evict_small", batch=3, kv_heads=4, dim=64, capacity=1500, length=1357, ragged=0.4, keep=257,
             recent=64, dtype="f32"),
        # the 64K-token cache cut to a quarter
        dict(_EVICT, name="evict_64k", capacity=65536, length=65521, keep=16384, recent=1024),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_LIMIT = {}


def _size(case):
    """(scores or kept rows, bytes) that bound what a pass costs."""
    if case["op"] == "evict":
        rows = case["batch"] * case["kv_heads"] * case["capacity"] * case["dim"]
    else:
        rows = case["batch"] * case["q_heads"] * _q_len(case) * case["capacity"]
    return rows, case["batch"] * case["kv_heads"] * case["capacity"] * case["dim"] * _es(case)


def _fits(case):
    if not _LIMIT:
        for c in listed():
            a, b = _size(c)
            la, lb = _LIMIT.get(c["op"], (0, 0))
            _LIMIT[c["op"]] = (max(a, la), max(b, lb))
    a, b = _size(case)
    la, lb = _LIMIT[case["op"]]
    return a <= la and b <= lb


def draw(rng):
    op = rng.choice(["tree", "chunk", "accumulate", "evict"])
    while True:
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        group = rng.choice([1, 2, 3, 4, 4, 6, 8])
        dim = rng.choice([64, 128, 128, 128, 256])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        if dtype == "f32" and dim == 256:
            dim = 128
        capacity = _log_int(rng, 16, 65536)
        length = max(1, int(capacity * rng.uniform(0.6, 1.0)))
        base = dict(batch=_log_int(rng, 1, 8), kv_heads=kv_heads, dim=dim, capacity=capacity, length=length,
                    ragged=rng.choice([0.0, round(rng.uniform(0.05, 0.9), 2)]), dtype=dtype)
        if op == "evict":
            keep = _log_int(rng, 1, length)
            case = dict(_EVICT, **base, keep=keep, recent=rng.choice([0, rng.randint(0, keep)]))
        elif op == "tree":
            case = dict(_TREE, **base, q_heads=kv_heads * group, nodes=_log_int(rng, 1, 128),
                        paged=rng.random() < 0.4, cap=rng.choice([0.0, 0.0, 30.0]))
            if case["paged"]:
                case["capacity"] = (capacity + PAGE - 1) // PAGE * PAGE
        else:
            q_len = rng.choice([1, _log_int(rng, 1, length), _log_int(rng, 1, length)])
            if op == "chunk":
                case = dict(_CHUNK, **base, q_heads=kv_heads * group, q_len=q_len, causal=rng.random() < 0.85,
                            prefix=rng.choice([0, rng.randint(1, length)]),
                            document=rng.choice([0, 0, _log_int(rng, 8, 4096)]), slopes=rng.random() < 0.3,
                            cap=rng.choice([0.0, 30.0, 50.0]))
            else:
                case = dict(_ACC, **base, q_heads=kv_heads * group, q_len=q_len, cap=rng.choice([0.0, 0.0, 50.0]))
        if _fits(case):
            return case


def _q_len(case):
    return case["nodes"] if case["op"] == "tree" else case["q_len"]


def _lengths(case):
    """Tokens of each batch row, from ``length`` down by the share ``ragged``."""
    B = case["batch"]
    return np.array([max(1, int(case["length"] * (1.0 - case["ragged"] * b / B))) for b in range(B)], np.int64)


def _documents(case):
    """Document of each token: pieces of uneven length around ``document``, the last five tokens padding (-1)."""
    S, step = case["capacity"], case["document"]
    sizes = np.maximum(1, np.array([step // 2, step + step // 2, step - step // 4, step + step // 4]))
    reps = np.resize(sizes, S // int(sizes.min()) + 1)
    ids = np.repeat(np.arange(len(reps)), reps)[:S]
    if S > 64:
        ids[-5:] = -1
    return ids


def _prefixes(case):
    return np.array([max(0, case["prefix"] - 37 * b) for b in range(case["batch"])], np.int64)


def _tree_parents(case, rng):
    n = case["nodes"]
    return np.array([-1] + [int(rng.integers(max(-1, t - 6), t)) for t in range(1, n)], np.int64)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = _dt(case)
    B, S, H, D = case["batch"], case["capacity"], case["kv_heads"], case["dim"]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    st = dict(case=case, lengths=lengths)
    # keys with a common direction per head that a few tokens (the first ones, and one in fifty) have more of: the
    # heavy hitters that real attention shows
    lean = 0.5 * randn(1, 1, H, D)
    heavy = (torch.rand((B, S, 1, 1), generator=g, device="cuda") < 0.02).float()
    heavy[:, :4] = 1.0
    keys = (randn(B, S, H, D) + heavy * lean).to(dt)
    values = randn(B, S, H, D).to(dt)
    if case["op"] == "evict":
        w = torch.exp(2.0 * randn(B, H, S) - 2.0)
        st.update(keys=keys, values=values, weights=(w * 64.0).round() / 64.0)  # many small equal values
        return st
    Hq, Sq = case["q_heads"], _q_len(case)
    st["q"] = (randn(B, Sq, Hq, D) + lean.repeat_interleave(Hq // H, dim=2)).to(dt)
    if case["op"] == "tree":
        rng = np.random.default_rng(int(seed))
        mask = np.zeros((B, Sq, Sq), bool)
        for b in range(B):
            for t, p in enumerate(_tree_parents(case, rng)):
                if p >= 0:
                    mask[b, t] = mask[b, p]
                mask[b, t, t] = True
        st["tree_mask"] = torch.tensor(mask, device="cuda")
        st["draft_keys"] = randn(B, Sq, H, D).to(dt)
        st["draft_values"] = randn(B, Sq, H, D).to(dt)
        if case["paged"]:  # the pages of all rows shuffled in one pool
            n = S // PAGE
            table = torch.randperm(B * n, generator=g, device="cuda")
            keys_pool, values_pool = torch.empty_like(keys), torch.empty_like(values)
            keys_pool.view(B * n, PAGE, H, D)[table] = keys.view(B * n, PAGE, H, D)
            values_pool.view(B * n, PAGE, H, D)[table] = values.view(B * n, PAGE, H, D)
            st["block_table"] = table.view(B, n).to(torch.int32)
            keys, values = keys_pool.view(B * S, H, D), values_pool.view(B * S, H, D)
    elif case["op"] == "chunk":
        if case["document"]:
            st["documents"] = torch.tensor(_documents(case), dtype=torch.int32, device="cuda").repeat(B, 1)
        if case["prefix"]:
            st["prefix"] = torch.tensor(_prefixes(case), dtype=torch.int32, device="cuda")
        if case["slopes"]:
            st["slopes"] = 2.0 ** (-8.0 * (torch.arange(Hq, device="cuda") + 1) / Hq)
    else:
        st["weights"] = torch.rand((B, H, S), generator=g, device="cuda")
    st.update(keys=keys, values=values)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    if own:
        return _run_own(st)
    op = st["case"]["op"]
    if op == "tree":
        return _plain_tree(st)
    if op == "chunk":
        return _plain_chunk(st)
    if op == "accumulate":
        return _plain_accumulate(st)
    return _plain_evict(st)


def _run_own(st):
    import orthocache_b200 as oc
    c = st["case"]
    if c["op"] == "tree":
        return oc.tree_attention(st["q"], st["keys"], st["values"], st["draft_keys"], st["draft_values"],
                                 st["tree_mask"], st["lengths"], block_table=st.get("block_table"), cap=c["cap"])
    if c["op"] == "chunk":
        return oc.chunk_attention(st["q"], st["keys"], st["values"], st["lengths"], causal=c["causal"],
                                  prefix=st.get("prefix"), documents=st.get("documents"), slopes=st.get("slopes"),
                                  cap=c["cap"])
    if c["op"] == "accumulate":
        return oc.accumulate_attention(st["q"], st["keys"], st["values"], st["weights"], st["lengths"], cap=c["cap"])
    return oc.evict_tokens(st["keys"], st["values"], st["weights"], c["keep"], recent=c["recent"],
                           lengths=st["lengths"])


def _heads_first(x, H):
    """(B, N, H * G, D) -> (B, H, G * N, D) in float32, rows of a KV head ordered (g, n)."""
    B, N, Hq, D = x.shape
    return x.float().view(B, N, H, Hq // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, (Hq // H) * N, D)


def _heads_back(x, N, dtype):
    B, H, R, D = x.shape
    return x.view(B, H, R // N, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, H * (R // N), D).to(dtype)


def _capped(s, cap):
    return cap * torch.tanh(s / cap) if cap > 0 else s


def _softmax(s, visible):
    """Softmax over the visible keys; a row that sees none is all zeros."""
    s = torch.where(visible, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _plain_tree(st):
    c, q, keys, values = st["case"], st["q"], st["keys"], st["values"]
    B, T, H, D = c["batch"], c["nodes"], c["kv_heads"], c["dim"]
    S, G = c["capacity"], c["q_heads"] // c["kv_heads"]
    if c["paged"]:
        table = st["block_table"].long()
        keys = keys.view(-1, PAGE, H, D)[table].view(B, S, H, D)
        values = values.view(-1, PAGE, H, D)[table].view(B, S, H, D)
    keys = torch.cat([keys, st["draft_keys"]], 1).float()
    values = torch.cat([values, st["draft_values"]], 1).float()
    s = _capped(_heads_first(q, H) @ keys.permute(0, 2, 3, 1) * D ** -0.5, c["cap"]).view(B, H, G, T, S + T)
    past = (torch.arange(S, device=q.device) < st["lengths"][:, None])[:, None, :].expand(B, T, S)
    visible = torch.cat([past, st["tree_mask"]], 2)[:, None, None]
    p = _softmax(s, visible).view(B, H, G * T, S + T)
    return _heads_back(p @ values.transpose(1, 2), T, q.dtype)


def _plain_chunk_weights(st, causal, prefix, documents, slopes):
    c, q = st["case"], st["q"]
    B, N, H, S, D = c["batch"], c["q_len"], c["kv_heads"], c["capacity"], c["dim"]
    G = c["q_heads"] // H
    s = _heads_first(q, H) @ st["keys"].float().permute(0, 2, 3, 1) * D ** -0.5
    s = _capped(s, c["cap"]).view(B, H, G, N, S)
    lengths = st["lengths"].long()
    j = torch.arange(S, device=q.device)
    pos = lengths[:, None] - N + torch.arange(N, device=q.device)  # (B, N)
    if slopes is not None:
        far = (pos[:, :, None] - j).abs().float()
        s = s - slopes.view(1, H, G, 1, 1) * far[:, None, None]
    visible = (j < lengths[:, None])[:, None, :] & (pos >= 0)[:, :, None]
    if causal:
        back = j <= pos[:, :, None]
        if prefix is not None:
            back = back | (j < prefix[:, None])[:, None, :]
        visible = visible & back
    if documents is not None:
        mine = torch.gather(documents, 1, pos.clamp(min=0))
        visible = visible & (mine[:, :, None] == documents[:, None, :]) & (mine >= 0)[:, :, None]
    return _softmax(s, visible[:, None, None]).view(B, H, G * N, S)


def _plain_chunk(st):
    c = st["case"]
    p = _plain_chunk_weights(st, c["causal"], st.get("prefix"), st.get("documents"), st.get("slopes"))
    return _heads_back(p @ st["values"].float().transpose(1, 2), c["q_len"], st["q"].dtype)


def _plain_accumulate(st):
    p = _plain_chunk_weights(st, True, None, None, None)
    out = _heads_back(p @ st["values"].float().transpose(1, 2), st["case"]["q_len"], st["q"].dtype)
    return out, st["weights"] + p.sum(2)


def _plain_evict(st):
    c, w = st["case"], st["weights"]
    B, H, S, keep = c["batch"], c["kv_heads"], c["capacity"], c["keep"]
    n = st["lengths"].long().view(B, 1, 1)
    pos = torch.arange(S, device=w.device)
    rank = torch.where(pos >= n, -math.inf, torch.where(pos >= n - c["recent"], math.inf, w))
    index = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    left = torch.clamp(n, max=keep)
    real = torch.arange(keep, device=w.device) < left
    at = index.transpose(1, 2)[..., None].expand(B, keep, H, c["dim"])
    there = real.expand(B, H, keep).transpose(1, 2)[..., None]
    zero = torch.zeros((), dtype=st["keys"].dtype, device=w.device)
    keys = torch.where(there, torch.gather(st["keys"], 1, at), zero)
    values = torch.where(there, torch.gather(st["values"], 1, at), zero)
    weights = torch.where(real, torch.gather(w, 2, index), 0.0)
    return keys, values, weights, torch.where(real, index, -1).to(torch.int32), left.view(B).to(torch.int32)


# ---------------------------------------------------------------------------
# the definition in 64 bits, one (batch row, KV head) at a time
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(case, st)
    B, N, H, D = case["batch"], _q_len(case), case["kv_heads"], case["dim"]
    G = case["q_heads"] // H
    q = st["q"].view(B, N, H, G, D)
    out = torch.zeros((B, N, H, G, D), dtype=torch.float64, device=q.device)
    sums = None
    if case["op"] == "accumulate":
        sums = st["weights"].double().clone()
    for b, n in enumerate(_lengths(case).tolist()):
        for h in range(H):
            if case["op"] == "tree":
                if case["paged"]:
                    t = st["block_table"][b].long()
                    at = (t[:, None] * PAGE + torch.arange(PAGE, device=t.device)).reshape(-1)[:n]
                    k, v = st["keys"][at, h], st["values"][at, h]
                else:
                    k, v = st["keys"][b, :n, h], st["values"][b, :n, h]
                k = torch.cat([k, st["draft_keys"][b, :, h]]).double()
                v = torch.cat([v, st["draft_values"][b, :, h]]).double()
                hidden = torch.zeros((N, n + N), dtype=torch.bool, device=k.device)
                hidden[:, n:] = ~st["tree_mask"][b]
            else:
                k, v = st["keys"][b, :n, h].double(), st["values"][b, :n, h].double()
                hidden = _exact_hidden(case, st, b, n)
            for lo in range(0, N, 512):
                rows = q[b, lo:lo + 512, h].double()  # (rows, G, D)
                z = torch.einsum("ngd,sd->gns", rows, k) / math.sqrt(D)
                if case["cap"] > 0:
                    z = (z / case["cap"]).tanh_().mul_(case["cap"])
                if case.get("slopes"):
                    i = n - N + lo + torch.arange(rows.shape[0], device=k.device, dtype=torch.float64)
                    far = (i[:, None] - torch.arange(n, device=k.device, dtype=torch.float64)).abs_()
                    z -= st["slopes"].double().view(H, G)[h].view(G, 1, 1) * far
                hide = hidden[lo:lo + 512]
                z.masked_fill_(hide, -math.inf)
                p = torch.exp(z - torch.logsumexp(z, -1, keepdim=True)).masked_fill_(hide, 0.0)
                out[b, lo:lo + 512, h] = torch.einsum("gns,sd->ngd", p, v)
                if sums is not None:
                    sums[b, h, :n] += p.sum((0, 1))
    out = out.view(B, N, H * G, D)
    return out if sums is None else (out, sums)


def _exact_hidden(case, st, b, n):
    N = case["q_len"]
    i = (n - N + torch.arange(N, device="cuda"))[:, None]
    j = torch.arange(n, device="cuda")[None, :]
    hidden = (i < 0) | torch.zeros_like(j, dtype=torch.bool)
    if case.get("causal", True):
        ahead = j > i
        if case.get("prefix"):
            ahead = ahead & (j >= int(_prefixes(case)[b]))
        hidden = hidden | ahead
    if case.get("document"):
        d = st["documents"][b]
        mine = d[i.clamp(min=0)]
        hidden = hidden | (mine != d[j]) | (mine < 0)
    return hidden


def _exact_evict(case, st):
    B, H, S, keep, recent = case["batch"], case["kv_heads"], case["capacity"], case["keep"], case["recent"]
    w = st["weights"].double().cpu().numpy()
    index = np.full((B, H, keep), -1, np.int64)
    lens = _lengths(case)
    for b in range(B):
        n = int(lens[b])
        for h in range(H):
            if n <= keep:
                pick = np.arange(n)
            else:
                old = np.lexsort((np.arange(n - recent), -w[b, h, :n - recent]))[:keep - recent]
                pick = np.concatenate([np.sort(old), np.arange(n - recent, n)])
            index[b, h, :len(pick)] = pick
    idx = torch.tensor(index, device="cuda")
    at = idx.clamp(min=0).transpose(1, 2)[..., None].expand(B, keep, H, case["dim"])
    real = (idx >= 0).transpose(1, 2)[..., None]
    keys = torch.gather(st["keys"].double(), 1, at) * real
    values = torch.gather(st["values"].double(), 1, at) * real
    weights = torch.gather(st["weights"].double(), 2, idx.clamp(min=0)) * (idx >= 0)
    left = torch.tensor(np.minimum(lens, keep), device="cuda")
    return keys, values, weights, idx.to(torch.int32), left.to(torch.int32)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _visible_pairs(case):
    """(query position, key) pairs that the masks leave, over the batch, and the keys that any query sees."""
    pairs = seen = 0
    for b, n in enumerate(_lengths(case).tolist()):
        if case["op"] == "tree":
            N = case["nodes"]
            pairs += N * n + N * (N + 1) // 2  # at most: every ancestor of a chain
            seen += n + N
            continue
        N = case["q_len"]
        i = np.arange(max(0, n - N), n)
        lo, hi = np.zeros_like(i), np.full_like(i, n - 1)
        if case.get("causal", True):
            hi = i.copy()
            if case.get("prefix"):
                hi = np.maximum(hi, min(n, int(_prefixes(case)[b])) - 1)
        if case.get("document"):
            d = _documents(case)[:n]
            ok = d[i] >= 0
            i, lo, hi = i[ok], lo[ok], hi[ok]
            first = np.searchsorted(np.where(d < 0, 1 << 30, d), d[i], side="left")
            last = np.searchsorted(np.where(d < 0, 1 << 30, d), d[i], side="right") - 1
            lo, hi = np.maximum(lo, first), np.minimum(hi, last)
        pairs += int(np.maximum(hi - lo + 1, 0).sum())
        seen += int(hi.max(initial=-1) - lo.min(initial=0)) + 1 if len(i) else 0
    return pairs, seen


def work(case):
    B, H, D, es = case["batch"], case["kv_heads"], case["dim"], _es(case)
    if case["op"] == "evict":
        kept = int(np.minimum(_lengths(case), case["keep"]).sum()) * H
        out_rows = B * H * case["keep"]
        scanned = int(_lengths(case).sum()) * H
        return {"bytes": 2 * (kept + out_rows) * D * es + scanned * 4 + out_rows * 8, "flops": scanned}
    pairs, seen = _visible_pairs(case)
    rows = B * _q_len(case) * case["q_heads"]
    nbytes = 2 * seen * H * D * es + 2 * rows * D * es
    flops = 4 * pairs * case["q_heads"] * D
    if case["op"] == "tree":
        nbytes += B * case["nodes"] ** 2
    if case["op"] == "accumulate":
        nbytes += 2 * B * H * case["capacity"] * 4
        flops += pairs * case["q_heads"]
    return {"bytes": nbytes, "flops": flops}
