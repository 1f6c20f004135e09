"""The attention and cache-eviction operators, as calls on inputs of the sizes they meet.

Three operators that a serving loop runs one after another:

* ``prompt``: attention over whole prompts (grouped heads, causal, dense with
  lengths and a key mask, or packed), its output and row log-sum-exp;
* ``cached``: attention of one token, or of a tree of drafted tokens, over a
  paged key/value cache, for one token with the accumulated weight of each key;
* ``evict``: eviction from such a cache by accumulated weight.

``run`` makes the plain form of each with elementary torch operations in
32 bits, or (``own``) the package's calls; ``exact`` restates the definitions in
64 bits.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _package():
    path = str(Path(__file__).resolve().parent.parent / "kv-block-mass_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kvblockmass_b200

    return kvblockmass_b200


def listed():
    return [
        # one user's long prompt at the Llama-3-8B attention shape
        {"name": "prompt_16k", "op": "prompt", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "lens": "16384", "packed": False, "causal": True, "mask": False},
        # a serving batch of prompts of very different lengths, packed one after another
        {"name": "prompt_packed", "op": "prompt", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128,
         "lens": "1 17 129 1000 3001 4044", "packed": True, "causal": True, "mask": False},
        # a padded batch of short fp16 prompts, one of them empty, some keys masked, no causality (an encoder)
        {"name": "prompt_padded_masked", "op": "prompt", "dtype": "fp16", "heads": 8, "kv_heads": 2, "dim": 64,
         "lens": "333 0 257 64", "packed": False, "causal": False, "mask": True},
        # the repository's benchmark shape in fp32: attention for numerical work
        {"name": "prompt_fp32", "op": "prompt", "dtype": "fp32", "heads": 8, "kv_heads": 2, "dim": 64,
         "lens": "2048", "packed": False, "causal": True, "mask": False},
        # a batch of users each decoding one token over a long paged cache, the weights of each key accumulated
        {"name": "token_batch", "op": "cached", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 32,
         "most": 8192, "least": 4097, "page": 16, "tokens": 1, "weights": True, "offsets": False},
        # one user decoding one token over a short cache: latency
        {"name": "token_short", "op": "cached", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 1,
         "most": 1000, "least": 1000, "page": 16, "tokens": 1, "weights": False, "offsets": False},
        # a wide tree of drafted tokens verified over long caches
        {"name": "tree_64_long", "op": "cached", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 4,
         "most": 32768, "least": 30001, "page": 64, "tokens": 64, "weights": False, "offsets": False},
        # a narrow fp16 tree over a cache that eviction thinned out: log offsets, pages that end inside a tile
        {"name": "tree_13_odd", "op": "cached", "dtype": "fp16", "heads": 8, "kv_heads": 2, "dim": 64, "batch": 7,
         "most": 3001, "least": 13, "page": 24, "tokens": 13, "weights": False, "offsets": True},
        # one token over caches already cut down to a budget: fp32, offsets of the sampled tail
        {"name": "token_fp32", "op": "cached", "dtype": "fp32", "heads": 8, "kv_heads": 2, "dim": 64, "batch": 8,
         "most": 2048, "least": 1024, "page": 2048, "tokens": 1, "weights": True, "offsets": True},
        # a batch of long caches cut to a quarter, every kv head by its own weights
        {"name": "evict_heads", "op": "evict", "dtype": "bf16", "kv_heads": 8, "dim": 128, "batch": 8, "most": 16384,
         "least": 12001, "page": 16, "budget": 4096, "shared": False},
        # one long cache, one choice for all heads (per-token mass of the prompt)
        {"name": "evict_shared", "op": "evict", "dtype": "bf16", "kv_heads": 8, "dim": 128, "batch": 1, "most": 32768,
         "least": 32768, "page": 64, "budget": 8192, "shared": True},
        # short fp32 caches, some within the budget already
        {"name": "evict_short", "op": "evict", "dtype": "fp32", "kv_heads": 2, "dim": 64, "batch": 3, "most": 300,
         "least": 60, "page": 16, "budget": 128, "shared": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["prompt", "cached", "evict"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 64, 128, 128, 96])
    if op == "prompt":
        n = rng.randint(1, 6)
        top = _log_int(rng, 1, 1024 if dtype == "fp32" else 4096)
        lens = [max(0, int(top * rng.random())) for _ in range(n - 1)] + [top]
        packed = rng.random() < 0.5
        return {"op": op, "dtype": dtype, "heads": kv_heads * rng.choice([1, 3, 4, 8]) if kv_heads < 8 else 32,
                "kv_heads": kv_heads, "dim": dim, "lens": " ".join(map(str, lens)), "packed": packed,
                "causal": rng.random() < 0.7, "mask": not packed and rng.random() < 0.4}
    most = _log_int(rng, 64, 16384)
    least = max(1, int(most * rng.random()))
    page = rng.choice([1, 8, 16, 24, 64, 100, 128, 256])
    if op == "cached":
        tokens = rng.choice([1, 1, 1, 2, 5, 16, 27, 64])
        return {"op": op, "dtype": dtype, "heads": kv_heads * rng.choice([1, 2, 4, 7]), "kv_heads": kv_heads, "dim": dim,
                "batch": _log_int(rng, 1, 32 if tokens < 16 else 6), "most": max(most, tokens),
                "least": max(least, tokens), "page": page, "tokens": tokens,
                "weights": tokens == 1 and rng.random() < 0.5, "offsets": rng.random() < 0.4}
    return {"op": op, "dtype": dtype, "kv_heads": kv_heads, "dim": dim, "batch": _log_int(rng, 1, 16), "most": most,
            "least": least, "page": page, "budget": max(48, int(most * rng.uniform(0.1, 0.9))),
            "shared": rng.random() < 0.4}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, d = _DTYPES[case["dtype"]], case["dim"]
    op = {"device": "cuda", "generator": g}
    if case["op"] == "prompt":
        lens = [int(x) for x in case["lens"].split()]
        hq, hkv, n, b = case["heads"], case["kv_heads"], max(lens), len(lens)
        rows = (sum(lens), 1) if case["packed"] else (b, n)
        # heads of different sharpness: q and k ~ N(0, 1) times a scale of U(0.5, 2) per head
        sq = 0.5 + 1.5 * torch.rand(hq, 1, **op)
        sk = 0.5 + 1.5 * torch.rand(hkv, 1, **op)
        q = (torch.randn(*rows, hq, d, **op) * sq).to(dt)
        k = (torch.randn(*rows, hkv, d, **op) * sk).to(dt)
        v = torch.randn(*rows, hkv, d, **op).to(dt)
        st = {"case": case, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "longest": n}
        if case["packed"]:
            cu = [0]
            cu.extend(sum(lens[:i + 1]) for i in range(b))
            st["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
            st["q"], st["k"], st["v"] = q[:, 0], k[:, 0], v[:, 0]
        else:
            st["q"], st["k"], st["v"] = (t.transpose(1, 2).contiguous() for t in (q, k, v))
            st["mask"] = (torch.rand(n, **op) > 0.1) if case["mask"] else None
        return st
    b, hkv, page = case["batch"], case["kv_heads"], case["page"]
    per = -(-case["most"] // page)
    lens = torch.randint(case["least"], case["most"] + 1, (b,), dtype=torch.int32, **op)
    st = {"case": case, "lens": lens, "table": torch.randperm(b * per, **op).to(torch.int32).reshape(b, per),
          "k": (torch.randn(b * per, page, hkv, d, **op) * (0.5 + 1.5 * torch.rand(hkv, 1, **op))).to(dt),
          "v": torch.randn(b * per, page, hkv, d, **op).to(dt)}
    length = per * page
    if case["op"] == "evict":
        # accumulated weights: a heavy tail, and many keys that nothing ever attended to (ties at zero)
        w = torch.exp(3.0 * torch.randn(b, 1 if case["shared"] else hkv, length, **op) - 4.0)
        st["weights"] = torch.where(torch.rand(w.shape, **op) < 0.3, torch.zeros_like(w), w)
        return st
    t, hq = case["tokens"], case["heads"]
    st["q"] = torch.randn(b, hq, t, d, **op).to(dt)
    if t > 1:
        # a random tree: node u's parent is one of the nodes before it
        parent = (torch.rand(b, t, **op) * torch.arange(t, device="cuda")).long()
        tree = torch.eye(t, dtype=torch.bool, device="cuda").repeat(b, 1, 1)
        for u in range(1, t):
            tree[:, u] |= tree[torch.arange(b, device="cuda"), parent[:, u]]
        st["tree"] = tree
    if case["weights"]:
        st["weights"] = torch.rand(b, hkv, length, **op)
        st["weights_out"] = torch.zeros(b, hkv, length, device="cuda")
    if case["offsets"]:
        # -log of inclusion probabilities: 0 for certain tokens, up to about 4 for the sampled tail
        p = torch.rand(b, hkv, length, **op)
        st["offsets"] = torch.where(p < 0.5, torch.zeros_like(p), 4.0 * torch.rand(p.shape, **op))
    return st


def _prompt_plain(st):
    c = st["case"]
    q, k, v, lens, n = st["q"], st["k"], st["v"], st["lens"].long(), st["longest"]
    at = torch.arange(n, device=q.device)
    inside = at[None] < lens[:, None]  # [B, N]
    if c["packed"]:
        first = st["cu"][:-1].long()
        where = (first[:, None] + at[None]).clamp(max=max(q.shape[0] - 1, 0))
        q, k, v = (t[where].transpose(1, 2) for t in (q, k, v))  # [B, H, N, D]
    b, hq, _, d = q.shape
    hkv = k.shape[1]
    keep = inside[:, None, :].expand(b, n, n)
    if c["causal"]:
        keep = keep & (at[None, :] <= at[:, None])
    if st.get("mask") is not None:
        keep = keep & st["mask"]
    keep = keep & inside[:, :, None]
    kf, vf = k.float(), torch.where(inside[:, None, :, None], v.float(), 0.0)
    s = torch.matmul(q.float().reshape(b, hkv, -1, d), kf.transpose(2, 3)).mul_(1.0 / math.sqrt(d))
    s = s.view(b, hkv, -1, n, n).masked_fill_(~keep[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    s = s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, hkv, -1, n), vf).view(b, hkv, -1, n, d)
    o = torch.where(total > 0, o / total, 0.0).reshape(b, hq, n, d).to(st["q"].dtype)
    lse = (top + total.log())[..., 0].reshape(b, hq, n)
    if c["packed"]:
        return {"out": o.transpose(1, 2)[inside], "lse": lse.transpose(1, 2)[inside].t().contiguous()}
    return {"out": o, "lse": lse}


def _paged_rows(cache, table):
    """[num_pages, page, H, D] through [B, pages] as [B, H, pages * page, D]."""
    rows = cache[table.long()]
    return rows.reshape(table.shape[0], -1, *cache.shape[2:]).transpose(1, 2)


def _cached_plain(st):
    q, lens = st["q"], st["lens"].long()
    b, hq, t, d = q.shape
    k, v = _paged_rows(st["k"], st["table"]).float(), _paged_rows(st["v"], st["table"]).float()
    hkv, n = k.shape[1], k.shape[2]
    at = torch.arange(n, device=q.device)
    inside = at[None] < lens[:, None]
    keep = inside[:, None, :].expand(b, t, n)
    if t > 1:
        draft = at[None] - (lens[:, None] - t)  # which drafted token sits in a slot
        seen = torch.gather(st["tree"], 2, draft.clamp(0, t - 1)[:, None, :].expand(b, t, n))
        keep = keep & ((draft < 0)[:, None] | seen)
    s = torch.matmul(q.float().reshape(b, hkv, -1, d), k.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).view(b, hkv, -1, t, n)
    if "offsets" in st:
        s = s + st["offsets"][:, :, None, None]
    s = s.masked_fill_(~keep[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total)
    out = torch.matmul(p.view(b, hkv, -1, n), v).reshape(b, hq, t, d).to(q.dtype)
    res = {"out": out, "lse": (top + total.log())[..., 0].reshape(b, hq, t)}
    if "weights" in st:
        res["weights"] = torch.where(inside[:, None], st["weights"] + p.sum((2, 3)), st["weights_out"])
    return res


_SINKS, _RECENCY = 4, 32


def _evict_plain(st):
    c, lens, w = st["case"], st["lens"].long(), st["weights"]
    b, hw, n = w.shape
    budget = c["budget"]
    at = torch.arange(n, device=w.device)
    length = lens[:, None, None]
    inside = at < length
    kept_always = (at < _SINKS) | (at >= length - _RECENCY) | (length <= budget)
    # order: the kept ones, then by weight; equal ones by index; what is not in the cache last
    key = torch.where(torch.isnan(w), -math.inf, w)
    order = torch.argsort(key, dim=-1, descending=True, stable=True)
    group = torch.where(inside, torch.where(kept_always, 0, 1), 2).expand(b, hw, n)
    by_group = torch.argsort(torch.gather(group, 2, order), dim=-1, stable=True)
    order = torch.gather(order, 2, by_group)
    if budget > n:
        order = torch.cat([order, order.new_full((b, hw, budget - n), n)], -1)
    new_lens = lens.clamp(max=budget)
    live = torch.arange(budget, device=w.device) < new_lens[:, None, None]
    slots = torch.where(live, order[..., :budget], n).sort(-1).values  # ascending, the rest behind
    source = slots.clamp(max=n - 1)
    hkv, d = st["k"].shape[2], st["k"].shape[3]
    rows = source.expand(b, hkv, budget)
    page = st["k"].shape[1]
    pages = torch.gather(st["table"].long()[:, None].expand(b, hkv, -1), 2, rows // page)
    heads = torch.arange(hkv, device=w.device)[None, :, None]
    k, v = st["k"][pages, rows % page, heads], st["v"][pages, rows % page, heads]
    shut = ~live[..., None].expand(b, hkv, budget, d)
    return {"k": k.masked_fill(shut, 0).transpose(1, 2), "v": v.masked_fill(shut, 0).transpose(1, 2),
            "seq_lens": new_lens.int(), "kept": torch.where(live, slots, -1).int(),
            "weights": torch.where(live, torch.gather(w, 2, source), 0.0)}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"prompt": _prompt_plain, "cached": _cached_plain, "evict": _evict_plain}[op](state)
    kb = _package()
    st, c = state, state["case"]
    if op == "prompt":
        if c["packed"]:
            out, lse = kb.attention_varlen(st["q"], st["k"], st["v"], st["cu"], st["longest"], causal=c["causal"])
        else:
            out, lse = kb.attention_b200(st["q"], st["k"], st["v"], attn_mask=st["mask"], causal=c["causal"],
                                         seq_lens=st["lens"])
        return {"out": out, "lse": lse}
    if op == "cached":
        res = kb.attention_cached(st["q"], st["k"], st["v"], st["table"], st["lens"], tree_mask=st.get("tree"),
                                  log_offsets=st.get("offsets"), weights=st.get("weights"),
                                  weights_out=st.get("weights_out"))
        return dict(zip(("out", "lse", "weights"), res))
    e = kb.evict_cache(st["k"], st["v"], st["table"], st["lens"], st["weights"], c["budget"], n_sinks=_SINKS,
                       recency=_RECENCY)
    return {"k": e.k, "v": e.v, "seq_lens": e.seq_lens, "kept": e.kept, "weights": e.weights}


def work(case):
    es, d = _BYTES[case["dtype"]], case["dim"]
    if case["op"] == "prompt":
        lens = [int(x) for x in case["lens"].split()]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        rows = sum(lens)
        return {"bytes": rows * (2 * case["heads"] + 2 * case["kv_heads"]) * d * es + 4 * rows * case["heads"],
                "flops": 4 * d * case["heads"] * pairs}
    b, hkv = case["batch"], case["kv_heads"]
    keys = b * (case["most"] + case["least"]) // 2
    if case["op"] == "cached":
        rows = b * case["heads"] * case["tokens"]
        extra = (8 if case["weights"] else 0) + (4 if case["offsets"] else 0)
        return {"bytes": keys * hkv * (2 * d * es + extra) + rows * (2 * d * es + 4),
                "flops": 4 * d * (case["heads"] // hkv) * case["tokens"] * hkv * keys}
    kept = b * min(case["budget"], (case["most"] + case["least"]) // 2)
    hw = 1 if case["shared"] else hkv
    return {"bytes": 4 * keys * hw + kept * hkv * 4 * d * es + kept * hw * 8, "flops": keys * hw}


def _softmax64(x, v):
    """Row softmax of x [..., R, N] (masked: -inf) times v [..., N, D], and the row log-sum-exp, in 64 bits."""
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(torch.isinf(lse), 0.0, lse)[..., None])
    return p, p @ v, lse


def exact(case, seed):
    st = prepare(case, seed)
    f64, dev = torch.float64, "cuda"
    if case["op"] == "prompt":
        q, k, v = st["q"], st["k"], st["v"]
        lens = [int(x) for x in case["lens"].split()]
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros(q.shape, dtype=f64, device=dev)
        rows_of = (q.shape[1], q.shape[0]) if case["packed"] else tuple(q.shape[:3])
        lse = torch.full(rows_of, -math.inf, dtype=f64, device=dev)
        first = 0
        for b, n in enumerate(lens):
            for h in range(case["heads"]):
                for r0 in range(0, n, 4096):  # query rows in pieces: the scores of one piece fit easily
                    r1 = min(n, r0 + 4096)
                    if case["packed"]:
                        qq = q[first + r0:first + r1, h]
                        kk, vv = k[first:first + n, h // group], v[first:first + n, h // group]
                    else:
                        qq, kk, vv = q[b, h, r0:r1], k[b, h // group, :n], v[b, h // group, :n]
                    x = qq.to(f64) @ kk.to(f64).T / math.sqrt(case["dim"])
                    if case["causal"]:
                        x = x.masked_fill(torch.ones(r1 - r0, n, dtype=torch.bool, device=dev).triu(r0 + 1), -math.inf)
                    if st.get("mask") is not None:
                        x = x.masked_fill(~st["mask"][:n], -math.inf)
                    _, o, l = _softmax64(x, vv.to(f64))
                    if case["packed"]:
                        out[first + r0:first + r1, h], lse[h, first + r0:first + r1] = o, l
                    else:
                        out[b, h, r0:r1], lse[b, h, r0:r1] = o, l
            first += n
        return {"out": out, "lse": lse}
    lens, page, table = st["lens"].tolist(), case["page"], st["table"].long()
    hkv, d = case["kv_heads"], case["dim"]
    if case["op"] == "evict":
        w, budget = st["weights"].to(f64).cpu(), case["budget"]
        hw = w.shape[1]
        k = torch.zeros(len(lens), budget, hkv, d, dtype=f64, device=dev)
        v, wout = torch.zeros_like(k), torch.zeros(len(lens), hw, budget, dtype=f64, device=dev)
        for b, n in enumerate(lens):
            for g in range(hkv):
                if hw > 1 or g == 0:
                    if n <= budget:
                        kept = list(range(n))
                    else:
                        row = w[b, g].tolist()
                        free = sorted(range(_SINKS, n - _RECENCY), key=lambda i: (-row[i], i))
                        kept = sorted([*range(_SINKS), *free[:budget - _SINKS - _RECENCY], *range(n - _RECENCY, n)])
                    kept = torch.tensor(kept, device=dev, dtype=torch.long)
                    wout[b, g, :len(kept)] = w[b, g].to(dev)[kept]
                pages = table[b, kept // page]
                k[b, :len(kept), g] = st["k"][pages, kept % page, g].to(f64)
                v[b, :len(kept), g] = st["v"][pages, kept % page, g].to(f64)
        return {"k": k, "v": v, "seq_lens": None, "kept": None, "weights": wout}
    b, hq, t, _ = st["q"].shape
    group = hq // hkv
    out = torch.zeros(b, hq, t, d, dtype=f64, device=dev)
    lse = torch.zeros(b, hq, t, dtype=f64, device=dev)
    weights = st["weights_out"].to(f64) if "weights" in st else None
    for i, n in enumerate(lens):
        pos = torch.arange(n, device=dev)
        pages = table[i, pos // page]
        kk, vv = (st[x][pages, pos % page].to(f64).transpose(0, 1) for x in "kv")  # [Hkv, n, D]
        x = st["q"][i].to(f64).reshape(hkv, group * t, d) @ kk.transpose(1, 2) / math.sqrt(d)
        if "offsets" in st:
            x = x + st["offsets"][i, :, :n].to(f64)[:, None]
        if t > 1:
            shut = torch.cat([torch.zeros(t, n - t, dtype=torch.bool, device=dev), ~st["tree"][i]], 1)
            x = x.view(hkv, group, t, n).masked_fill(shut, -math.inf).view(hkv, group * t, n)
        p, o, l = _softmax64(x, vv)
        out[i], lse[i] = o.reshape(hq, t, d), l.reshape(hq, t)
        if weights is not None:
            weights[i, :, :n] = st["weights"][i, :, :n].to(f64) + p.sum(1)
    res = {"out": out, "lse": lse}
    if weights is not None:
        res["weights"] = weights
    return res
