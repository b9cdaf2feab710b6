"""Workloads of the paged-cache operators: page transfer (append, gather), attention of new tokens over a paged
cache (causal, with an optional sliding window and sinks), the attention weight that it leaves on every cached
token, and eviction by that weight.

`own = False` computes each operator in its plain form (elementary torch operations in 32 bits, rounded once);
`own = True` calls kvforge_b200.PagedKVCache. A case is a dict of plain values; its sequence lengths follow from
the case alone, its values from the seed."""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # one decoding step of a batch writes one token per sequence: nothing but latency
        dict(name="append_decode", op="append", dtype="float16", heads=8, dim=128, page=64, seqs=64, new_min=1,
             new_max=1, old_min=100, old_max=4000, mix=1),
        # a 16384-token prompt of the streaming workload goes into the cache at once
        dict(name="append_prompt", op="append", dtype="bfloat16", heads=8, dim=128, page=64, seqs=1, new_min=16384,
             new_max=16384, old_min=0, old_max=0, mix=2),
        # a finished 32k sequence leaves its pages for the codec, as [heads, tokens, dim]
        dict(name="gather_32k", op="gather", dtype="float16", heads=8, dim=128, page=64, seqs=1, old_min=32768,
             old_max=32768, mix=3),
        # one token of one sequence on a short cache: the latency of a single user
        dict(name="decode_one", op="attend", dtype="float16", heads=8, group=4, dim=128, page=64, seqs=1, new_min=1,
             new_max=1, old_min=2047, old_max=2047, window=0, sinks=0, lse=True, mix=4),
        # a batch of users in the middle of their answers, lengths from nothing to 16k, small pages
        dict(name="decode_batch", op="attend", dtype="bfloat16", heads=8, group=8, dim=128, page=16, seqs=64,
             new_min=1, new_max=1, old_min=0, old_max=16383, window=0, sinks=0, lse=False, mix=5),
        # a chunk of a long prompt on the 32k cache of the 8-head workload: the matrix products count
        dict(name="chunk_32k", op="attend", dtype="float16", heads=8, group=4, dim=128, page=64, seqs=1,
             new_min=2048, new_max=2048, old_min=30720, old_max=30720, window=0, sinks=0, lse=False, mix=6),
        # chunks and single tokens in one batch, a window of 1000 with 4 sinks, odd group, narrow heads
        dict(name="mixed_window", op="attend", dtype="bfloat16", heads=4, group=5, dim=64, page=32, seqs=12,
             new_min=1, new_max=1023, old_min=0, old_max=12000, window=1000, sinks=4, lse=False, mix=7),
        # the codec's own f32 caches: a chunk in full precision
        dict(name="chunk_f32", op="attend", dtype="float32", heads=32, group=1, dim=128, page=64, seqs=1,
             new_min=500, new_max=500, old_min=1548, old_max=1548, window=0, sinks=0, lse=True, mix=8),
        # a prompt's last chunk, its attention recorded for eviction
        dict(name="track_chunk", op="track", dtype="bfloat16", heads=8, group=4, dim=128, page=64, seqs=2,
             new_min=1000, new_max=1030, old_min=7000, old_max=7200, window=0, sinks=0, lse=False, mix=9),
        # a decoding step whose weights replace the old ones (eviction by the latest query)
        dict(name="track_decode", op="track", dtype="float16", heads=8, group=8, dim=128, page=64, seqs=16,
             new_min=1, new_max=1, old_min=3000, old_max=16000, window=0, sinks=0, lse=False, mix=10),
        # one layer of a few sequences back to a small budget
        dict(name="evict_small", op="evict", dtype="float16", heads=8, dim=128, page=64, layers=1, seqs=4,
             old_min=1000, old_max=1200, budget=777, recent=64, sinks=4, mix=11),
        # every layer of a 32k sequence down to a quarter
        dict(name="evict_32k", op="evict", dtype="bfloat16", heads=8, dim=128, page=64, layers=16, seqs=1,
             old_min=32768, old_max=32768, budget=8192, recent=1024, sinks=4, mix=12),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm (lo may be 0)."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))) - 1)))


def draw(rng):
    op = rng.choice(["append", "gather", "attend", "attend", "attend", "attend", "track", "track", "evict", "evict"])
    dtype = rng.choice(["float16", "bfloat16", "float16", "bfloat16", "float32"])
    c = dict(op=op, dtype=dtype, heads=rng.choice([1, 2, 4, 8, 8, 16, 32]), dim=rng.choice([32, 64, 80, 96, 128, 128]),
             page=rng.choice([16, 32, 64, 128]), mix=rng.randrange(1 << 20))
    if op == "append":
        c["seqs"] = _log(rng, 1, 96)
        hi = max(1, 16384 * 8 // (c["seqs"] * c["heads"]))
        c["new_max"] = _log(rng, 1, hi)
        c["new_min"] = rng.choice([c["new_max"], 0, max(1, c["new_max"] // 2)])
        c["old_max"] = _log(rng, 0, 8000)
        c["old_min"] = rng.choice([0, c["old_max"] // 2])
    elif op == "gather":
        c["seqs"] = 1
        c["old_min"] = c["old_max"] = _log(rng, 1, 32768 * 8 // c["heads"])
    elif op in ("attend", "track"):
        c["group"] = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
        while c["heads"] * c["group"] > 128:
            c["group"] = max(1, c["group"] // 2)
        if rng.random() < 0.5:  # single tokens, or a few (drafts)
            c["seqs"] = _log(rng, 1, 128)
            c["new_max"] = rng.choice([1, 1, 1, 2, 4, 7])
            c["new_min"] = 1
            c["old_max"] = _log(rng, 1, min(65536, 64 * 16384 * 8 // (c["seqs"] * c["heads"])))
        else:  # chunks, the cost bounded by the largest listed one's pairs
            c["seqs"] = _log(rng, 1, 12)
            c["new_max"] = _log(rng, 16, 4096)
            c["new_min"] = rng.choice([c["new_max"], 1, max(1, c["new_max"] // 2)])
            pairs = 2048 * 32768 * 32 // (4 if dtype == "float32" else 1)
            while c["seqs"] * c["new_max"] * c["new_max"] * c["heads"] * c["group"] > pairs:
                c["new_max"] = max(1, c["new_max"] // 2)
                c["new_min"] = min(c["new_min"], c["new_max"])
            c["old_max"] = _log(rng, 0, min(32768, max(0, pairs // (c["seqs"] * c["new_max"] * c["heads"] * c["group"])
                                                       - c["new_max"])))
        c["old_min"] = rng.choice([c["old_max"], 0, c["old_max"] // 2])
        c["window"] = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
        c["sinks"] = rng.choice([0, 4, 33]) if c["window"] else 0
        c["lse"] = rng.random() < 0.3
    else:
        c["layers"] = rng.choice([1, 1, 2, 8])
        c["seqs"] = _log(rng, 1, 16)
        c["old_max"] = _log(rng, 2, min(65536, 16 * 32768 * 8 // (c["layers"] * c["seqs"] * c["heads"])))
        c["old_min"] = rng.choice([c["old_max"], c["old_max"] // 2])
        c["budget"] = max(1, int(c["old_max"] * rng.uniform(0.1, 0.9)))
        c["sinks"] = min(rng.choice([0, 4]), c["budget"])
        c["recent"] = rng.choice([0, min(c["budget"] - c["sinks"], _log(rng, 1, 1024))])
    return c


def _lengths(case):
    """(tokens cached before the call, new tokens) of every sequence; the first one has the longest of both."""
    rng = random.Random(case["mix"])
    n = case["seqs"]
    old = [case["old_max"] if i == 0 else _log(rng, case["old_min"], case["old_max"]) for i in range(n)]
    if "new_max" not in case:
        return old, [0] * n
    return old, [case["new_max"] if i == 0 else _log(rng, case["new_min"], case["new_max"]) for i in range(n)]


def _rows(gen, shape, dtype, scale=1.0):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return (x if scale == 1.0 else x.mul_(scale)).to(dtype)


def prepare(case, seed):
    """Page pools filled with a cache whose pages are scattered, the page table, and the call's new rows."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype, H, D, page = case["op"], DTYPES[case["dtype"]], case["heads"], case["dim"], case["page"]
    layers = case.get("layers", 1)
    old, new = _lengths(case)
    total = [a + b for a, b in zip(old, new)]
    need = [-(-t // page) for t in total]
    used = sum(need)
    spare = -(-case["budget"] // page) * case["seqs"] if op == "evict" else 0
    order = np.random.RandomState(seed % (1 << 31)).permutation(used)
    first = np.concatenate([[0], np.cumsum(need)]).astype(np.int64)
    shape = (layers, used + spare, H, page)
    # keys have a few channels that are larger than the others, as caches do
    wide = torch.ones(D, device="cuda")
    wide[torch.randperm(D, generator=gen, device="cuda")[:4]] = 4.0
    keys = torch.empty(shape + (D,), dtype=dtype, device="cuda")
    values = torch.empty(shape + (D,), dtype=dtype, device="cuda")
    for l in range(layers):
        keys[l] = (torch.randn(shape[1:] + (D,), generator=gen, device="cuda") * wide).to(dtype)
        values[l] = _rows(gen, shape[1:] + (D,), dtype)
    # accumulated weight: heavy-tailed, a fifth of the tokens never looked at (ties)
    weights = torch.exp(2.0 * torch.randn(shape, generator=gen, device="cuda"))
    weights *= torch.rand(shape, generator=gen, device="cuda") > 0.2
    if spare:
        for x in (keys, values, weights):
            x[:, used:] = 0
    s = dict(case, first=first, old=old, new=new, total=total, keys=keys, values=values, weights=weights, used=used)
    maxp = max(1, max(need))
    table = np.zeros((len(old), maxp), np.int64)
    for b in range(len(old)):
        table[b, :need[b]] = order[first[b]:first[b + 1]]
    s["table"] = torch.from_numpy(table).cuda()
    s["len"] = torch.tensor(total, device="cuda")
    N = sum(new)
    # which sequence a new token belongs to, and its place there
    seq = np.repeat(np.arange(len(new)), new)
    at = np.concatenate([np.arange(c) for c in new]) if N else np.zeros(0, np.int64)
    s["seq"], s["at"] = torch.from_numpy(seq).cuda(), torch.from_numpy(at).cuda()
    s["new_len"] = torch.tensor(new, device="cuda")
    if op == "append":
        s["new_keys"], s["new_values"] = _rows(gen, (N, H, D), dtype), _rows(gen, (N, H, D), dtype)
    if op in ("attend", "track"):
        s["query"] = _rows(gen, (N, H * case["group"], D), dtype)
    if own:
        import kvforge_b200 as K
        cache = K.PagedKVCache(used + spare, H, D, page_size=page, num_layers=layers, dtype=dtype)
        cache.keys.copy_(keys)
        cache.values.copy_(values)
        cache.weights.copy_(weights)
        seqs = [cache.add(length=old[b], pages=[int(p) for p in order[first[b]:first[b + 1]]]) for b in range(len(old))]
        s.update(cache=cache, seqs=seqs, keys=None, values=None, weights=None)
        if op in ("attend", "track"):
            s["batch"] = cache.extend(seqs, new, query_heads=H * case["group"], window=case["window"],
                                      sinks=case["sinks"])
        elif op == "append":
            s["batch"] = cache.extend(seqs, new)
    return s


def run(s):
    return (_own if own else _plain)[s["op"]](s)


# ---- the framework's operators -----------------------------------------------------------------------------------
def _own_append(s):
    c = s["cache"]
    c.append(s["batch"], s["new_keys"], s["new_values"])
    return {"keys": c.keys, "values": c.values, "weights": c.weights}


def _own_gather(s):
    kv = s["cache"].gather(s["seqs"][0])
    return {"keys": kv.keys_tensor, "values": kv.values_tensor}


def _own_attend(s):
    if s["lse"]:
        out, lse = s["cache"].attend(s["batch"], s["query"], return_lse=True)
        return {"out": out, "lse": lse}
    return {"out": s["cache"].attend(s["batch"], s["query"])}


def _own_track(s):
    out = s["cache"].attend(s["batch"], s["query"], decay=0.0)
    return {"out": out, "weights": s["cache"].weights}


def _own_evict(s):
    c = s["cache"]
    e = c.evict(s["seqs"], s["budget"], recent=s["recent"], sinks=s["sinks"], keep_source=True)
    # the branches' pages are the ones that were free
    u = s["used"]
    r = {"kept": e.kept, "keys": c.keys[:, u:], "values": c.values[:, u:], "weights": c.weights[:, u:]}
    c.free(e.seqs)
    return r


_own = {"append": _own_append, "gather": _own_gather, "attend": _own_attend, "track": _own_track, "evict": _own_evict}


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _slots(s, seq, pos):
    """(page, row) of places `pos` of sequences `seq`."""
    return s["table"][seq, pos // s["page"]], pos % s["page"]


def _plain_append(s):
    pos = s["len"][s["seq"]] - s["new_len"][s["seq"]] + s["at"]
    p, r = _slots(s, s["seq"], pos)
    s["keys"][0][p, :, r] = s["new_keys"]
    s["values"][0][p, :, r] = s["new_values"]
    s["weights"][0][p, :, r] = 0.0
    return {"keys": s["keys"], "values": s["values"], "weights": s["weights"]}


def _lined(pool, table):
    """[B, H, tokens (padded to whole pages), ...] of a layer's pages."""
    x = pool[table].transpose(1, 2)
    return x.reshape(x.shape[:2] + (x.shape[2] * x.shape[3],) + x.shape[4:])


def _plain_gather(s):
    T = s["total"][0]
    return {"keys": _lined(s["keys"][0], s["table"])[0, :, :T].contiguous(),
            "values": _lined(s["values"][0], s["table"])[0, :, :T].contiguous()}


def _plain_scores(s):
    """Scores [B, H, group, queries, tokens] in 32 bits, -inf where a query does not see a token; and V."""
    H, G, D = s["heads"], s["group"], s["dim"]
    k, v = (_lined(s[n][0], s["table"]).float() for n in ("keys", "values"))
    B, T = k.shape[0], k.shape[2]
    C = max(s["new"])
    q = torch.zeros((B, C, H, G, D), device="cuda")
    q[s["seq"], s["at"]] = s["query"].reshape(-1, H, G, D).float()
    q = q.permute(0, 2, 3, 1, 4).reshape(B, H, G * C, D)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(B, H, G, C, T)
    a = (s["len"] - s["new_len"])[:, None] + torch.arange(C, device="cuda")
    j = torch.arange(T, device="cuda")
    see = j <= a[..., None]
    if s["window"]:
        see &= (j > a[..., None] - s["window"]) | (j < s["sinks"])
    see &= (torch.arange(C, device="cuda") < s["new_len"][:, None])[..., None]
    x.masked_fill_(~see[:, None, None], float("-inf"))
    v.masked_fill_((j >= s["len"][:, None])[:, None, :, None], 0.0)
    return x, v


def _plain_softmax(x):
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    p = x.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    return p, l, (m + torch.log(l)).squeeze(-1)


def _plain_out(s, p, l, v):
    B, H, G, C, T = p.shape
    o = torch.matmul(p.view(B, H, G * C, T), v).view(B, H, G, C, -1) / torch.where(l == 0, 1.0, l)
    o = o.permute(0, 3, 1, 2, 4)[s["seq"], s["at"]]
    return o.reshape(o.shape[0], H * G, -1).to(s["query"].dtype)


def _plain_attend(s):
    x, v = _plain_scores(s)
    p, l, lse = _plain_softmax(x)
    out = {"out": _plain_out(s, p, l, v)}
    if s["lse"]:
        lse = lse.permute(0, 3, 1, 2)[s["seq"], s["at"]]
        out["lse"] = lse.reshape(lse.shape[0], -1)
    return out


def _plain_track(s):
    x, v = _plain_scores(s)
    p, l, _ = _plain_softmax(x)
    out = _plain_out(s, p, l, v)
    w = (p / torch.where(l == 0, 1.0, l)).sum((2, 3))  # [B, H, tokens]
    B, H, T = w.shape
    j = torch.arange(T, device="cuda")
    b, j = torch.nonzero((j < s["len"][:, None]) & (s["new_len"] > 0)[:, None], as_tuple=True)
    p, r = _slots(s, b, j)
    s["weights"][0][p, :, r] = w[b, :, j]
    return {"out": out, "weights": s["weights"]}


def _plain_evict(s):
    L, B, H, page, N = s["layers"], s["seqs"], s["heads"], s["page"], s["budget"]
    w = torch.stack([_lined(x, s["table"]) for x in s["weights"]])  # [L, B, H, tokens]
    T = w.shape[-1]
    j = torch.arange(T, device="cuda")
    n = s["len"][:, None]
    always = (j < s["sinks"]) | (j >= n - s["recent"])
    rank = torch.where(always[:, None], float("inf"), w)
    rank = torch.where((j < n)[:, None], rank, -1.0)
    kept = torch.argsort(rank, dim=-1, descending=True, stable=True)[..., :N]
    n = n[:, :, None]  # a sequence that the budget holds keeps all its tokens
    kept = torch.where(kept < n, kept, T).sort(-1).values
    pad = N - kept.shape[-1]
    kept = torch.nn.functional.pad(kept, (0, pad), value=T)
    there = kept < n
    l, b, h, i = torch.nonzero(there, as_tuple=True)
    p, r = _slots(s, b, kept[l, b, h, i])
    np_ = -(-N // page)
    np_b = -(-torch.minimum(s["len"], torch.full_like(s["len"], N)) // page)
    at = torch.cumsum(np_b, 0) - np_b  # pages are handed out in order
    to_p, to_r = at[b] + i // page, i % page
    out = {"kept": torch.where(there, kept, -1).to(torch.int32)}
    for name in ("keys", "values", "weights"):
        x = s[name]
        y = torch.zeros((L, np_ * B) + x.shape[2:], dtype=x.dtype, device="cuda")
        y[l, to_p, h, to_r] = x[l, p, h, r]
        out[name] = y
    return out


_plain = {"append": _plain_append, "gather": _plain_gather, "attend": _plain_attend, "track": _plain_track,
          "evict": _plain_evict}


# ---- what one pass cannot do without ---------------------------------------------------------------------------------
def _pairs(old, new, window, sinks):
    """(query, token) pairs that are seen, and tokens that any query sees."""
    a = old + np.arange(new, dtype=np.int64)  # positions of the queries
    if not window:
        return int((a + 1).sum()), old + new if new else 0
    lo = np.maximum(0, a - window + 1)
    seen = a + 1 - lo + np.minimum(sinks, lo)
    if not new:
        return 0, 0
    first = max(0, old - window + 1)
    return int(seen.sum()), old + new - first + min(sinks, first)


def work(case):
    e = DTYPES[case["dtype"]].itemsize
    op, H, D = case["op"], case["heads"], case["dim"]
    old, new = _lengths(case)
    if op == "append":
        return {"bytes": sum(new) * H * (4 * D * e + 4), "flops": 0}
    if op == "gather":
        return {"bytes": sum(old) * H * 4 * D * e, "flops": 0}
    if op == "evict":
        kept = sum(min(n, case["budget"]) for n in old)
        return {"bytes": case["layers"] * H * (sum(old) * 4 + kept * (4 * D * e + 4 + 4)), "flops": 0}
    p = [_pairs(a, c, case["window"], case["sinks"]) for a, c in zip(old, new)]
    pairs, tokens = sum(x[0] for x in p), sum(x[1] for x in p)
    Hq = H * case["group"]
    b = tokens * H * 2 * D * e + sum(new) * Hq * 2 * D * e + (sum(new) * Hq * 4 if case["lse"] else 0)
    f = pairs * Hq * 4 * D
    if op == "track":
        b += sum(a + c for a, c in zip(old, new) if c) * H * 4
        f += pairs * Hq
    return {"bytes": b, "flops": f}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] not in ("attend", "track"):
        return None  # nothing is computed, only moved: the outputs are equal or wrong
    was = globals()["own"]
    globals()["own"] = False
    try:
        s = prepare(case, seed)
    finally:
        globals()["own"] = was
    H, G, D, page = case["heads"], case["group"], case["dim"], case["page"]
    N = sum(s["new"])
    out = torch.zeros((N, H * G, D), dtype=torch.float64, device="cuda")
    lse = torch.full((N, H * G), float("-inf"), dtype=torch.float64, device="cuda")
    weights = s["weights"].double()
    row = 0
    for b, (n, c) in enumerate(zip(s["total"], s["new"])):
        pages = s["table"][b, :-(-n // page)]
        for h in range(H):
            if not c:
                continue
            k = s["keys"][0, pages, h].reshape(-1, D)[:n].double()
            v = s["values"][0, pages, h].reshape(-1, D)[:n].double()
            total = torch.zeros(pages.numel() * page, dtype=torch.float64, device="cuda")
            for i0 in range(0, c, 1024):
                i1 = min(c, i0 + 1024)
                a = torch.arange(n - c + i0, n - c + i1, device="cuda")[:, None]
                j = torch.arange(n, device="cuda")[None]
                hidden = j > a
                if case["window"]:
                    hidden |= (a - j >= case["window"]) & (j >= case["sinks"])
                for g in range(h * G, h * G + G):
                    q = s["query"][row + i0:row + i1, g].double()
                    x = (q @ k.T / D ** 0.5).masked_fill(hidden, float("-inf"))
                    z = torch.logsumexp(x, 1)
                    p = torch.exp(x - z[:, None])
                    out[row + i0:row + i1, g] = p @ v
                    lse[row + i0:row + i1, g] = z
                    total[:n] += p.sum(0)
            w = weights[0, pages, h].reshape(-1)
            w[:n] = total[:n]
            weights[0, pages, h] = w.view(-1, page)
        row += c
    if case["op"] == "track":
        return {"out": out, "weights": weights}
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
