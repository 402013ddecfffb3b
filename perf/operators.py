"""Measured cases of the attention-layer operators around the paged cache.

Three operators, each in its plain form (elementary torch operations in 32 bits) and, with
``own`` set, as the calls a user makes of ``lmserve_b200.ops``:

* ``norm``: the norm of every query and key head, the rotary embedding and the cache write of one layer;
* ``paged``: attention of a batch over its pages of one layer's cache (decode steps and causal prefill chunks);
* ``prefix``: the same for a batch whose requests share long prefixes, held once in the cache.

Lengths are spread evenly between a case's bounds, so that a case's work is the same for every
seed; which request has which length, the pages and all values come from the seed.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of an interactive user: the launch is all there is
        dict(name="norm one token", kind="norm", tokens=1, heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16", max_pos=8192, padded=0, key_out=False),
        # a full decode batch, some slots of it padding
        dict(name="norm decode batch", kind="norm", tokens=256, heads=28, kv_heads=4, head_dim=128, block=16, dtype="bf16", max_pos=32768, padded=9, key_out=False),
        # one prefill step at the scheduler's token limit
        dict(name="norm prefill step", kind="norm", tokens=8192, heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16", max_pos=8192, padded=0, key_out=False),
        # an odd chunk of small heads whose rotated keys are wanted outside the cache as well
        dict(name="norm odd chunk", kind="norm", tokens=1023, heads=16, kv_heads=4, head_dim=64, block=16, dtype="fp16", max_pos=4096, padded=5, key_out=True),
        # one interactive user in mid-conversation
        dict(name="decode one request", kind="paged", batch=1, q_lo=0, q_hi=0, past_lo=4097, past_hi=4097, heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16", lse=False),
        # a full decode batch of ragged contexts, from a request without any key to long ones
        dict(name="decode ragged batch", kind="paged", batch=256, q_lo=0, q_hi=0, past_lo=0, past_hi=4000, heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16", lse=False),
        # one rank's single key head under tensor parallelism
        dict(name="decode one-head shard", kind="paged", batch=512, q_lo=0, q_hi=0, past_lo=200, past_hi=1500, heads=8, kv_heads=1, head_dim=128, block=16, dtype="bf16", lse=False),
        # a chunked prefill step: four prompts, some with an earlier chunk in the cache
        dict(name="prefill chunks", kind="paged", batch=4, q_lo=1000, q_hi=3000, past_lo=0, past_hi=2000, heads=28, kv_heads=4, head_dim=128, block=16, dtype="bf16", lse=True),
        # a few requests behind a short system prompt
        dict(name="prefix small", kind="prefix", groups=1, batch=4, q_lo=0, q_hi=0, prefix_lo=1000, prefix_hi=1000, past_lo=1, past_hi=50, heads=16, kv_heads=4, head_dim=64, block=16, dtype="fp16", lse=False),
        # a decode batch behind one long system prompt
        dict(name="prefix full batch", kind="prefix", groups=1, batch=256, q_lo=0, q_hi=0, prefix_lo=8192, prefix_hi=8192, past_lo=1, past_hi=512, heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16", lse=False),
        # several prompts in service at once, one of them of length zero
        dict(name="prefix groups", kind="prefix", groups=8, batch=120, q_lo=0, q_hi=0, prefix_lo=0, prefix_hi=4000, past_lo=16, past_hi=1000, heads=28, kv_heads=4, head_dim=128, block=16, dtype="bf16", lse=False),
        # new user turns, several tokens each, appended behind a shared prompt
        dict(name="prefix new turns", kind="prefix", groups=1, batch=32, q_lo=1, q_hi=64, prefix_lo=4096, prefix_hi=4096, past_lo=0, past_hi=200, heads=32, kv_heads=8, head_dim=128, block=16, dtype="fp16", lse=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _geometry(rng):
    heads, kv_heads = rng.choice([(32, 8), (28, 4), (16, 4), (8, 1), (14, 2), (6, 6)])
    return dict(heads=heads, kv_heads=kv_heads, head_dim=rng.choice([64, 128, 128]), block=rng.choice([16, 16, 16, 8, 32, 64, 12]), dtype=rng.choice(["bf16", "bf16", "fp16"]))


def _draw(rng):
    kind = rng.choice(["norm", "paged", "paged", "prefix", "prefix"])
    g = _geometry(rng)
    if kind == "norm":
        tokens = _log(rng, 1, 8192)
        return dict(kind=kind, tokens=tokens, max_pos=_log(rng, 2048, 32768), padded=rng.choice([0, 0, tokens // 20]), key_out=rng.random() < 0.3, **g)
    lse = rng.random() < 0.3
    if kind == "paged":
        if rng.random() < 0.6:
            hi = _log(rng, 1, 8192)
            return dict(kind=kind, batch=_log(rng, 1, 512), q_lo=0, q_hi=0, past_lo=rng.randint(0, hi), past_hi=hi, lse=lse, **g)
        q_hi = _log(rng, 1, 3000)
        p_hi = _log(rng, 1, 4000)
        return dict(kind=kind, batch=_log(rng, 1, 16), q_lo=rng.randint(1, q_hi), q_hi=q_hi, past_lo=rng.randint(0, p_hi), past_hi=p_hi, lse=lse, **g)
    batch = _log(rng, 2, 256)
    pre, hi = _log(rng, 100, 8192), _log(rng, 1, 1000)
    q_hi = rng.choice([0, 0, _log(rng, 1, 64)])
    return dict(kind=kind, groups=rng.randint(1, min(8, batch)), batch=batch, q_lo=min(q_hi, 1), q_hi=q_hi, prefix_lo=rng.choice([pre, rng.randint(0, pre)]), prefix_hi=pre, past_lo=rng.randint(0, hi), past_hi=hi, lse=lse, **g)


def draw(rng):
    caps = {}
    for c in listed():
        w = work(c)
        top = caps.setdefault(c["kind"], [0, 0])
        top[0], top[1] = max(top[0], w["bytes"]), max(top[1], w["flops"])
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= caps[c["kind"]][0] and w["flops"] <= caps[c["kind"]][1] and _padded_keys(c) <= 2_300_000_000:
            return c


# ------------------------------------------------------------------------------- lengths
def _spread(n, lo, hi):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _lengths(c):
    """Per request: (new tokens, keys of its own, group), and the groups' prefix lengths."""
    n = c["batch"]
    q = _spread(n, c["q_lo"], c["q_hi"]) if c["q_hi"] else [1] * n
    past = _spread(n, c["past_lo"], c["past_hi"])
    past = past[n // 2:] + past[: n // 2]  # the longest past is not the longest prompt's
    keys = [p + (k if c["q_hi"] else 0) for p, k in zip(past, q)]
    groups = c.get("groups", 0)
    return q, keys, [i * groups // n for i in range(n)] if groups else [0] * n, _spread(groups, c["prefix_lo"], c["prefix_hi"]) if groups else []


def _padded_keys(c):
    """Elements of the keys in the plain form, where every request is padded to the longest."""
    if c["kind"] == "norm":
        return 0
    q, keys, _, prefix = _lengths(c)
    return len(q) * (max(keys) + max(prefix, default=0)) * max(c["kv_heads"] * c["head_dim"], c["heads"] * max(q))


def work(case):
    c = case
    H, K, D = c["heads"], c["kv_heads"], c["head_dim"]
    if c["kind"] == "norm":
        T = c["tokens"]
        moved = 2 * T * (H + K) * D + 2 * (T - c["padded"]) * K * D + T * 2 * D  # q and k in and out, v in and out, the tables' rows
        return {"bytes": 2 * (moved + (T * K * D if c["key_out"] else 0)) + 16 * T, "flops": 8 * T * (H + K) * D}
    q, keys, group, prefix = _lengths(c)
    T = sum(q)
    pairs = sum(prefix[g] * n for g, n in zip(group, q)) if prefix else 0
    for n, k in zip(q, keys):
        pairs += n * k - n * (n - 1) // 2 if c["q_hi"] else k
    read = sum(keys) + sum(prefix)
    return {"bytes": 2 * (2 * T * H * D + 2 * read * K * D) + 4 * (read // c["block"]), "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dt, dev = case, DTYPES[case["dtype"]], "cuda"
    rng = np.random.default_rng([seed, 77])
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    H, K, D, bs = c["heads"], c["kv_heads"], c["head_dim"], c["block"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * scale).to(dt)

    def ids(a, kind=torch.int32):
        return torch.tensor(np.asarray(a), device=dev).to(kind)

    s = {"case": dict(c)}
    if c["kind"] == "norm":
        T = c["tokens"]
        blocks = -(-T // bs) + 3
        qkv = normal(T, (H + 2 * K) * D, scale=1.5)  # the projection's output: three strided views of it
        s["q"], s["k"], s["v"] = qkv[:, : H * D], qkv[:, H * D: (H + K) * D], qkv[:, (H + K) * D:]
        s["q_weight"], s["k_weight"] = normal(D, scale=0.2) + 1, normal(D, scale=0.2) + 1
        freqs = torch.arange(c["max_pos"], device=dev, dtype=torch.float64)[:, None] * 500000.0 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
        s["cos_sin"] = torch.cat((freqs.cos(), freqs.cos(), freqs.sin(), freqs.sin()), 1).to(dt)
        s["positions"] = ids(rng.integers(0, c["max_pos"], T))
        slots = rng.permutation(blocks * bs)[:T]
        slots[rng.permutation(T)[: c["padded"]]] = -1
        s["slots"] = ids(slots, torch.int64)
        s["cache"] = normal(blocks, 2, bs, K, D)
        return s

    q, keys, group, prefix = _lengths(c)
    if c["kind"] == "paged":  # the groups of the others are neighbours in the batch: only lengths move
        order = rng.permutation(c["batch"])
        q, keys = [q[i] for i in order], [keys[i] for i in order]
    else:
        for g in range(c["groups"]):
            at = [i for i, x in enumerate(group) if x == g]
            order = rng.permutation(len(at))
            for name in (q, keys):
                name[at[0]: at[-1] + 1] = [name[at[i]] for i in order]
    pages = [-(-k // bs) for k in keys + prefix]
    total = sum(pages)
    pool = total + total // 8 + 2
    table = rng.permutation(pool)[:total]
    cut = sum(pages[: len(keys)])

    def arrays(lengths, table):
        n = [-(-k // bs) for k in lengths]
        return ids(np.concatenate(([0], np.cumsum(n)))), ids(table), ids([k - (m - 1) * bs if m else 0 for k, m in zip(lengths, n)])

    T = sum(q)
    s["q"] = normal(T, H, D, scale=2.0)  # scores of spread 2: a few keys carry most of a row
    s["cache"] = normal(pool, 2, bs, K, D)
    s["kv_indptr"], s["kv_indices"], s["kv_last"] = arrays(keys, table[:cut])
    s["qo_indptr"] = ids(np.concatenate(([0], np.cumsum(q)))) if c["q_hi"] else None
    s["longest"] = (max(q), max(keys), max(prefix, default=0))
    if prefix:
        s["prefix_indptr"], s["prefix_indices"], s["prefix_last"] = arrays(prefix, table[cut:])
        s["group_indptr"] = ids([sum(x < g for x in group) for g in range(c["groups"] + 1)])
    return s


# ------------------------------------------------------------------------------- one pass
def run(state):
    s = state
    if own:
        return _own(s)
    if s["case"]["kind"] == "norm":
        return _plain_norm(s)
    return _plain_attention(s)


def _own(s):
    from lmserve_b200 import ops
    c = s["case"]
    if c["kind"] == "norm":
        got = ops.qk_norm_rotary_pos_emb_and_cache(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["positions"], s["cos_sin"], c["head_dim"],
                                                   s["cache"], s["slots"], eps=1e-6, return_key=c["key_out"])
        return (*got, s["cache"]) if c["key_out"] else (got, s["cache"])
    if c["kind"] == "paged":
        return ops.paged_attention(s["q"], s["cache"], s["kv_indptr"], s["kv_indices"], s["kv_last"], qo_indptr=s["qo_indptr"], return_lse=c["lse"])
    return ops.shared_prefix_attention(s["q"], s["cache"], s["prefix_indptr"], s["prefix_indices"], s["prefix_last"], s["kv_indptr"], s["kv_indices"], s["kv_last"],
                                       group_indptr=s["group_indptr"], qo_indptr=s["qo_indptr"], return_lse=c["lse"])


def _plain_norm(s):
    c = s["case"]
    T, D, dt, bs = c["tokens"], c["head_dim"], s["q"].dtype, c["block"]
    row = s["cos_sin"][s["positions"].long()].float()[:, None]
    cos, sin = row[..., :D], row[..., D:]

    def turned(x, weight):
        x = x.float().reshape(T, -1, D)
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
        half = torch.cat((-x[..., D // 2:], x[..., : D // 2]), -1)
        return (x * cos + half * sin).to(dt)

    q, k = turned(s["q"], s["q_weight"]), turned(s["k"], s["k_weight"])
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    s["cache"][at // bs, 0, at % bs] = k[keep]
    s["cache"][at // bs, 1, at % bs] = s["v"].reshape(k.shape)[keep]
    q, k = q.reshape(T, -1), k.reshape(T, -1)
    return (q, k, s["cache"]) if c["key_out"] else (q, s["cache"])


def _rows(indptr, indices, last, most, bs):
    """Slot ids [n, most] of every list of pages, and how many of them each has."""
    n = indptr[1:].long() - indptr[:-1].long()
    lengths = torch.where(n > 0, (n - 1) * bs + last.long(), torch.zeros_like(n))
    at = torch.arange(most, device=indptr.device)
    page = (indptr[:-1].long()[:, None] + at // bs).clamp(max=max(0, indices.numel() - 1))
    page = indices[page].long() if indices.numel() else torch.zeros_like(page)
    return page * bs + at % bs, lengths


def _plain_attention(s):
    c = s["case"]
    H, K, D, bs, dt = c["heads"], c["kv_heads"], c["head_dim"], c["block"], s["q"].dtype
    dev = s["q"].device
    q_most, k_most, p_most = s["longest"]
    slots, lengths = _rows(s["kv_indptr"], s["kv_indices"], s["kv_last"], k_most, bs)
    B, T = lengths.numel(), s["q"].shape[0]
    first = s["qo_indptr"].long() if s["qo_indptr"] is not None else torch.arange(B + 1, device=dev)
    of = torch.searchsorted(first[1:].contiguous(), torch.arange(T, device=dev), right=True)
    at = torch.arange(T, device=dev) - first[of]
    n_new = first[1:] - first[:-1]
    query = torch.zeros(B, q_most, H, D, device=dev)
    query[of, at] = s["q"].float()
    i, j = torch.arange(q_most, device=dev)[None, :, None], torch.arange(k_most, device=dev)[None, None]
    seen = (j < lengths[:, None, None]) & (j <= (lengths - n_new)[:, None, None] + i)
    if c["kind"] == "prefix":
        shared, p_len = _rows(s["prefix_indptr"], s["prefix_indices"], s["prefix_last"], p_most, bs)
        g = torch.searchsorted(s["group_indptr"][1:].long().contiguous(), torch.arange(B, device=dev), right=True)
        slots = torch.cat((shared[g], slots), 1)
        before = (torch.arange(p_most, device=dev)[None, None] < p_len[g][:, None, None]).expand(B, q_most, p_most)
        seen = torch.cat((before, seen), 2)
    page, entry = slots // bs, slots % bs
    keys = s["cache"][page, 0, entry].float().permute(0, 2, 3, 1)                         # [B, K, D, L]
    rows = query.reshape(B, q_most, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, -1, D)
    score = torch.matmul(rows, keys).mul_(1.0 / math.sqrt(D)).reshape(B, K, H // K, q_most, -1)
    del keys
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True) if score.shape[-1] else score.new_full((*score.shape[:-1], 1), float("-inf"))
    top = top.masked_fill(top == float("-inf"), 0.0)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    values = s["cache"][page, 1, entry].float().permute(0, 2, 1, 3)                       # [B, K, L, D]
    out = torch.matmul(score.reshape(B, K, -1, score.shape[-1]), values).reshape(B, K, H // K, q_most, D)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.permute(0, 3, 1, 2, 4).reshape(B, q_most, H, D)[of, at].to(dt)
    if not c["lse"]:
        return out
    lse = (total.log() + top)[..., 0].permute(0, 3, 1, 2).reshape(B, q_most, H)[of, at]
    return out, lse


# ------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if case["kind"] == "norm" else _exact_attention(s)


def _exact_norm(s):
    c = s["case"]
    D, E = c["head_dim"], c["head_dim"] // 2
    table = s["cos_sin"].double()[s["positions"].long()]

    def head(x, w):
        x = x.double().unflatten(1, (-1, D))
        x = w.double() * x / (x.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt()
        a, b = x[..., :E], x[..., E:]
        ca, cb, sa, sb = (table[:, None, i * E: (i + 1) * E] for i in range(4))
        return torch.cat((a * ca - b * sa, b * cb + a * sb), -1)

    q, k = head(s["q"], s["q_weight"]), head(s["k"], s["k_weight"])
    cache = s["cache"].double()
    flat = cache.transpose(1, 2).reshape(-1, 2, c["kv_heads"], D)                         # one row a slot
    keep = (s["slots"] >= 0).nonzero()[:, 0]
    flat[s["slots"][keep], 0] = k[keep]
    flat[s["slots"][keep], 1] = s["v"].double().unflatten(1, (-1, D))[keep]
    cache = flat.reshape(cache.shape[0], c["block"], 2, c["kv_heads"], D).transpose(1, 2)
    return (q.flatten(1), k.flatten(1), cache) if c["key_out"] else (q.flatten(1), cache)


def _exact_attention(s):
    c = s["case"]
    H, K, D, bs = c["heads"], c["kv_heads"], c["head_dim"], c["block"]

    def pages(indptr, indices, last):
        p, t, e = indptr.tolist(), indices.long(), last.tolist()
        return [(t[p[i]: p[i + 1]], max(0, (p[i + 1] - p[i] - 1) * bs + e[i])) for i in range(len(e))]

    def taken(what):
        t, n = what
        kv = s["cache"][t].double()                                                       # [pages, 2, bs, K, D]
        return kv[:, 0].reshape(-1, K, D)[:n], kv[:, 1].reshape(-1, K, D)[:n]

    mine = pages(s["kv_indptr"], s["kv_indices"], s["kv_last"])
    first = s["qo_indptr"].tolist() if s["qo_indptr"] is not None else list(range(len(mine) + 1))
    if c["kind"] == "prefix":
        shared = [taken(x) for x in pages(s["prefix_indptr"], s["prefix_indices"], s["prefix_last"])]
        bounds = s["group_indptr"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.full(s["q"].shape[:2], float("-inf"), dtype=torch.float64, device=s["q"].device)
    g = 0
    for b, what in enumerate(mine):
        keys, values = taken(what)
        a, z = first[b], first[b + 1]
        ahead = 0
        if c["kind"] == "prefix":
            while b >= bounds[g + 1]:
                g += 1
            keys, values, ahead = torch.cat((shared[g][0], keys)), torch.cat((shared[g][1], values)), shared[g][0].shape[0]
        if a == z or not keys.shape[0]:
            continue
        limit = ahead + what[1] - (z - a) + torch.arange(z - a, device=out.device)        # the last key each new token sees
        hidden = torch.arange(keys.shape[0], device=out.device)[None] > limit.clamp(min=ahead - 1)[:, None]
        for k in range(K):
            mineq = s["q"][a:z, k * (H // K): (k + 1) * (H // K)].double().transpose(0, 1)
            score = (mineq @ keys[:, k].T / D ** 0.5).masked_fill_(hidden, float("-inf"))
            total = torch.logsumexp(score, -1)
            weight = torch.exp(score - total[..., None]).nan_to_num_(0.0)
            out[a:z, k * (H // K): (k + 1) * (H // K)] = (weight @ values[:, k]).transpose(0, 1)
            lse[a:z, k * (H // K): (k + 1) * (H // K)] = total.T
    return (out, lse) if c["lse"] else out
