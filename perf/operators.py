"""The batched-decode operators, as cases to be timed and compared.

Four operators of a decode step over several sessions that share a paged
key-value cache:

  append   new tokens' K / V rows written into the pages (16-bit rows, or the
           affine group-64 codes of the quantized caches)
  attn     attention of one new token per session over its pages
  evict    the cache of every session cut to a budget by accumulated weight
  logits   per-row penalties, biases and allow masks

`run` computes them in plain torch operations while `own` is false and through
the framework's public calls while it is true.  `exact` computes them once
more in 64 bits, session by session.
"""
from __future__ import annotations

import math

import torch

own = False

GROUP = 64  # dims per scale and bias of the affine caches
BITS = {"bf16": (16, 16), "fp16": (16, 16), "k8v8": (8, 8), "k4v4": (4, 4), "k8v4": (8, 4)}
HEAVY = 1_000_000_000  # 16-bit bytes a drawn cache may hold; the largest listed one holds a little more


# --------------------------------------------------------------------------
# cases


def listed():
    return [
        # one chat session early in its reply: a call that only its latency counts for
        dict(name="attn one session 600", op="attn", kind="bf16", batch=1, hi=600, lo=600, hq=32, hkv=4, d=128, page=16,
             window=0, cap=0.0, sinks=False, weights=False),
        # one session over a whole long document, 8-bit cache: few rows, so the length has to be split
        dict(name="attn one session 131072 k8v8", op="attn", kind="k8v8", batch=1, hi=131072, lo=131072, hq=32, hkv=4,
             d=128, page=256, window=0, cap=0.0, sinks=True, weights=False),
        # a full server: 64 sessions of every length up to 16K
        dict(name="attn 64 sessions bf16", op="attn", kind="bf16", batch=64, hi=16384, lo=1, hq=32, hkv=4, d=128,
             page=64, window=0, cap=0.0, sinks=False, weights=False),
        # capped scores, sinks and a sliding window, 5 query heads a kv head, pages of 48
        dict(name="attn window cap sinks fp16", op="attn", kind="fp16", batch=24, hi=3001, lo=0, hq=20, hkv=4, d=64,
             page=48, window=513, cap=30.0, sinks=True, weights=False),
        # the step of a cache that is to be cut to a budget: attention that also accumulates its weights
        dict(name="attn weights bf16", op="attn", kind="bf16", batch=16, hi=8448, lo=300, hq=32, hkv=4, d=128, page=32,
             window=0, cap=0.0, sinks=False, weights=True),
        # the native path's mixed cache, a mid-size batch
        dict(name="attn 32 sessions k8v4", op="attn", kind="k8v4", batch=32, hi=8191, lo=17, hq=32, hkv=4, d=128,
             page=128, window=0, cap=0.0, sinks=False, weights=False),
        # every step of 64 sessions: one token each, quantized on append
        dict(name="append step k8v8", op="append", kind="k8v8", batch=64, hi=1, lo=1, start=4000, hkv=4, d=128, page=64),
        # a batch of prompts entering the cache
        dict(name="append prompts bf16", op="append", kind="bf16", batch=16, hi=8192, lo=5, start=100, hkv=4, d=128,
             page=32),
        # a running session's regular cut: one page of tokens over the budget
        dict(name="evict step bf16", op="evict", kind="bf16", batch=8, hi=4352, lo=4352, budget=4096, recent=256, hkv=4,
             d=128, page=32),
        # long prompts cut to an eighth
        dict(name="evict prompts k8v4", op="evict", kind="k8v4", batch=8, hi=65536, lo=30000, budget=8192, recent=512,
             hkv=4, d=128, page=128),
        # one session's logits in 32 bits, a short history
        dict(name="logits one row fp32", op="logits", kind="fp32", batch=1, vocab=151936, history=900, biases=8,
             mask=False),
        # a full server's logits: every row has its own rules, a grammar mask and a history of up to 4,096 ids
        dict(name="logits 64 rows bf16", op="logits", kind="bf16", batch=64, vocab=151936, history=4096, biases=64,
             mask=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "append", "evict", "logits"])
    if op == "logits":
        kind = rng.choice(["fp32", "bf16", "fp16"])
        return dict(op=op, kind=kind, batch=_log(rng, 1, 64), vocab=_log(rng, 1000, 200000), history=_log(rng, 1, 8192),
                    biases=rng.choice([0, 3, 37, 300]), mask=rng.random() < 0.5)
    kind = rng.choice(["bf16", "fp16", "k8v8", "k8v4", "k4v4"])
    hkv = rng.choice([1, 2, 3, 4, 8])
    d = rng.choice([64, 128, 128, 256]) if kind.startswith("k") else rng.choice([64, 80, 128, 128, 192, 256])
    page = rng.choice([1, 16, 24, 32, 64, 128, 256])
    row = 4 * hkv * d  # bytes of one token's K and V in 16 bits
    if op == "attn":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 1, max(2, min(131072, HEAVY // (row * batch))))
        return dict(op=op, kind=kind, batch=batch, hi=hi, lo=rng.choice([0, 1, hi]), hq=hkv * rng.choice([1, 2, 3, 4, 5, 8, 12, 16]),
                    hkv=hkv, d=d, page=page, window=rng.choice([0, 0, 0, 100, 4096]), cap=rng.choice([0.0, 0.0, 50.0]),
                    sinks=rng.random() < 0.5, weights=rng.random() < 0.3)
    if op == "append":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 1, max(2, min(16384, HEAVY // (4 * row * batch))))
        return dict(op=op, kind=kind, batch=batch, hi=hi, lo=rng.choice([0, 1, hi]), start=rng.choice([0, 1, 777, 5000]),
                    hkv=hkv, d=d, page=page)
    batch = _log(rng, 1, 24)
    hi = _log(rng, 64, max(65, min(100000, HEAVY // (2 * row * batch))))
    budget = _log(rng, 16, hi)
    return dict(op=op, kind=kind, batch=batch, hi=hi, lo=rng.choice([0, budget, hi]), budget=budget,
                recent=rng.choice([0, budget // 16, budget // 2]), hkv=hkv, d=d, page=page)


def _lengths(case):
    """The sessions' lengths: lo .. hi, evenly spread in the order of the
    fractional parts of i * golden ratio, so every seed has the same sum; the
    seed only permutes them."""
    n, lo, hi = case["batch"], case["lo"], case["hi"]
    lo = min(lo, hi)
    if n == 1:
        return [hi]
    return [lo + round((hi - lo) * ((0.5 + i * 0.6180339887498949) % 1.0)) for i in range(n - 1)] + [hi]


def _row_bytes(case):
    """Bytes of one token and kv head: K row + V row (codes, scales, biases)."""
    d = case["d"]
    return sum(d * 2 if b == 16 else d * b // 8 + 4 * (d // GROUP) for b in BITS[case["kind"]])


def work(case):
    if case["op"] == "logits":
        n = case["batch"] * case["vocab"]
        item = 4 if case["kind"] == "fp32" else 2
        extra = case["batch"] * (4 * case["history"] + 8 * case["biases"] + 20)
        return {"bytes": 2 * item * n + extra + (n / 8 if case["mask"] else 0), "flops": n}
    lengths = _lengths(case)
    hkv, d = case["hkv"], case["d"]
    tokens = sum(lengths)
    if case["op"] == "append":
        return {"bytes": tokens * hkv * (4 * d + _row_bytes(case)) + 8 * case["batch"], "flops": tokens * hkv * d * 2}
    if case["op"] == "attn":
        seen = sum(min(n, case["window"]) if case["window"] else n for n in lengths)
        io = 2 * 2 * case["batch"] * case["hq"] * d + 4 * sum(-(-n // case["page"]) for n in lengths)
        acc = 8 * tokens * hkv if case["weights"] else 0
        return {"bytes": seen * hkv * _row_bytes(case) + io + acc, "flops": 4 * seen * case["hq"] * d}
    moved = 0.0  # rows expected at or above the budget that survive: the protected ones, and a share of the others
    for n in lengths:
        if n > case["budget"]:
            r, b = min(case["recent"], case["budget"]), case["budget"]
            above = min(r, n - b)
            moved += above + (b - r) * max(0, n - b - above) / max(1, n - r)
    kept = sum(min(n, case["budget"]) for n in lengths)
    return {"bytes": hkv * (8 * tokens + 8 * kept + 2 * moved * _row_bytes(case)), "flops": hkv * tokens}


# --------------------------------------------------------------------------
# inputs


def _pool(g, kind, which, pages, hkv, page, d, fill):
    """One of the two pools: {"x": rows or codes, "s", "b": scales, biases}."""
    bits = BITS[kind][which]
    dev = g.device
    if bits == 16:
        dt = torch.float16 if kind == "fp16" else torch.bfloat16
        if not fill:
            return {"x": torch.zeros(pages, hkv, page, d, dtype=dt, device=dev)}
        return {"x": torch.randn(pages, hkv, page, d, dtype=dt, device=dev, generator=g)}
    if not fill:
        z = torch.zeros(pages, hkv, page, d // GROUP, dtype=torch.bfloat16, device=dev)
        return {"x": torch.zeros(pages, hkv, page, d * bits // 32, dtype=torch.int32, device=dev), "s": z, "b": z.clone()}
    x, s, b = _affine(torch.randn(pages, hkv, page, d, device=dev, generator=g), bits)
    return {"x": x, "s": s, "b": b}


def _table(g, lengths, page, spare=3):
    """Pages of every session in a shuffled order; unused entries -1."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g, device=g.device).to(torch.int32)
    width = max(1, max(need))
    at = torch.arange(width, device=g.device)[None, :]
    need_t = torch.tensor(need, device=g.device)[:, None]
    first = torch.cumsum(need_t, 0) - need_t
    table = torch.where(at < need_t, order[(first + at).clamp_max(total - 1)], torch.full_like(at, -1, dtype=torch.int32))
    return table.contiguous(), total


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    dev = g.device
    s = {"case": case}
    if case["op"] == "logits":
        B, V, n, m = case["batch"], case["vocab"], case["history"], case["biases"]
        dt = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[case["kind"]]
        s["logits"] = (torch.randn(B, V, device=dev, generator=g) * 3).to(dt)
        s["out"] = torch.empty(B, V, dtype=dt, device=dev)
        # token ids as text repeats them: few frequent ones, many rare ones
        u = torch.rand(B, n, device=dev, generator=g)
        s["history"] = (V * u ** 4).to(torch.int32).clamp_max(V - 1)
        s["history_len"] = torch.randint(n // 2, n + 1, (B,), device=dev, generator=g, dtype=torch.int32)
        s["prompt_len"] = (s["history_len"] * 0.4).to(torch.int32)
        s["repetition"] = 1.0 + 0.3 * torch.rand(B, device=dev, generator=g)
        s["frequency"] = 0.5 * torch.rand(B, device=dev, generator=g)
        s["presence"] = 0.5 * torch.rand(B, device=dev, generator=g)
        s["bias_ids"] = torch.randint(-1, V, (B, m), device=dev, generator=g, dtype=torch.int32) if m else None
        s["bias_values"] = 5 * torch.randn(B, m, device=dev, generator=g) if m else None
        words = (V + 31) // 32
        # a grammar allows few ids in most states and most ids inside free text
        some = torch.randint(-2**31, 2**31, (B, words), device=dev, generator=g, dtype=torch.int64)
        some &= torch.randint(-2**31, 2**31, (B, words), device=dev, generator=g, dtype=torch.int64)
        s["allow"] = some.to(torch.int32) if case["mask"] else None
        return s
    hkv, d, page, kind, B = case["hkv"], case["d"], case["page"], case["kind"], case["batch"]
    order = torch.randperm(B, generator=g, device=dev).tolist()
    own_lengths = _lengths(case)
    lengths = [own_lengths[i] for i in order]
    i32 = dict(dtype=torch.int32, device=dev)
    if case["op"] == "append":
        starts = [case["start"]] * B
        s["table"], pages = _table(g, [a + n for a, n in zip(starts, lengths)], page)
        s["k"], s["v"] = (_pool(g, kind, w, pages, hkv, page, d, False) for w in (0, 1))
        dt = torch.float16 if kind == "fp16" else torch.bfloat16
        total = sum(lengths)
        s["new_k"] = torch.randn(total, hkv, d, dtype=dt, device=dev, generator=g)
        s["new_v"] = torch.randn(total, hkv, d, dtype=dt, device=dev, generator=g)
        s["starts"] = torch.tensor(starts, **i32)
        s["cu"] = torch.tensor([sum(lengths[:i]) for i in range(B + 1)], **i32)
        return s
    s["lengths"] = torch.tensor(lengths, **i32)
    s["table"], pages = _table(g, lengths, page)
    s["k"], s["v"] = (_pool(g, kind, w, pages, hkv, page, d, True) for w in (0, 1))
    if case["op"] == "attn":
        dt = torch.float16 if kind == "fp16" else torch.bfloat16
        s["q"] = (2 * torch.randn(B, case["hq"], d, device=dev, generator=g)).to(dt)
        s["sinks"] = torch.randn(case["hq"], device=dev, generator=g).to(torch.bfloat16) if case["sinks"] else None
        if case["weights"]:
            s["weights"] = torch.rand(pages, hkv, page, device=dev, generator=g)
            s["weights_out"] = torch.zeros(pages, hkv, page, device=dev)
        return s
    # accumulated weights: a few heavy tokens, a long tail, and some that no query ever looked at
    w = torch.rand(pages, hkv, page, device=dev, generator=g) ** 6 * 8
    w[torch.rand(pages, hkv, page, device=dev, generator=g) < 0.1] = 0.0
    s["weights"] = w
    s["weights_out"] = torch.zeros_like(w)
    # positions: the slots' own, as before any earlier cut
    idx = torch.arange(s["table"].shape[1] * page, device=dev)
    pos = torch.zeros(pages, hkv, page, **i32)
    pg = s["table"][:, idx // page].long()
    ok = pg >= 0
    off = (idx % page)[None, :].expand_as(pg)
    pos[pg[ok], :, off[ok]] = idx[None, :].expand_as(pg)[ok].to(torch.int32)[:, None].expand(-1, hkv)
    s["positions"], s["positions_out"] = pos, torch.zeros_like(pos)
    s["keep_from"] = (s["lengths"] - case["recent"]).to(torch.int32)
    s["lengths_out"] = torch.zeros(B, **i32)
    return s


# --------------------------------------------------------------------------
# plain forms


def _affine(x, bits):
    """Affine group-64 quantisation: codes packed into 32-bit words, bf16
    scales and biases.  x fp32 [..., D]."""
    shape = x.shape
    w = x.reshape(*shape[:-1], shape[-1] // GROUP, GROUP)
    top, low = w.amax(-1, keepdim=True), w.amin(-1, keepdim=True)
    bins = torch.full((1,), float((1 << bits) - 1), device=x.device)  # a tensor: a true division, no reciprocal
    scale = ((top - low) / bins).clamp_min(1e-7)
    side = low.abs() > top.abs()
    scale = torch.where(side, scale, -scale)
    edge = torch.where(side, low, top)
    q0 = torch.round(edge / scale)
    scale = torch.where(q0 != 0, edge / q0, scale)
    bias = torch.where(q0 != 0, edge, torch.zeros_like(edge))
    codes = torch.round((w - bias) / scale).clamp(0, (1 << bits) - 1).to(torch.int32)
    per = 32 // bits
    words = codes.reshape(*shape[:-1], shape[-1] // per, per)
    shift = torch.arange(per, device=x.device, dtype=torch.int32) * bits
    words = (words << shift).sum(-1, dtype=torch.int32)
    return words, scale.squeeze(-1).to(torch.bfloat16), bias.squeeze(-1).to(torch.bfloat16)


def _values(pool, bits, pick, dt):
    """The rows that `pick` takes from a pool, as `dt` values [..., D]."""
    x = pick(pool["x"])
    if bits == 16:
        return x.to(dt)
    per = 32 // bits
    shift = torch.arange(per, device=x.device, dtype=torch.int32) * bits
    c = ((x[..., None] >> shift) & ((1 << bits) - 1)).reshape(*x.shape[:-1], -1, GROUP).to(dt)
    c = c * pick(pool["s"])[..., None].to(dt) + pick(pool["b"])[..., None].to(dt)
    return c.reshape(*x.shape[:-1], -1)


def _slots(s, n):
    """(page ids [B, n] with -1 as 0, offsets [n]) of slots 0 .. n - 1."""
    page = s["case"]["page"]
    idx = torch.arange(n, device=s["table"].device)
    return s["table"][:, idx // page].clamp_min(0).long(), idx % page, idx


def _attn(s):
    c = s["case"]
    hkv, d, kb, vb = c["hkv"], c["d"], *BITS[c["kind"]]
    B, n = c["batch"], max(1, c["hi"])
    pg, off, idx = _slots(s, n)
    K = _values(s["k"], kb, lambda t: t[pg, :, off], torch.float32)  # [B, n, hkv, d]
    q = s["q"].float().reshape(B, hkv, -1, d)
    x = torch.matmul(q, K.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    del K
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    L = s["lengths"].long()[:, None]
    seen = idx[None, :] < L
    if c["window"]:
        seen = seen & (idx[None, :] >= L - c["window"])
    x = x.masked_fill(~seen[:, None, None, :], float("-inf"))
    m = x.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].float().reshape(1, hkv, -1, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = torch.exp(x - m)
    del x
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - m)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    V = _values(s["v"], vb, lambda t: t[pg, :, off], torch.float32)
    V = V.masked_fill(~seen[:, :, None, None], 0.0)
    out = torch.matmul(p, V.permute(0, 2, 1, 3)).reshape(B, hkv * q.shape[2], d).to(s["q"].dtype)
    if not c["weights"]:
        return {"out": out}
    ok = idx[None, :] < L
    new = 0.98 * s["weights"][pg, :, off] + p.sum(2).permute(0, 2, 1)  # [B, n, hkv]
    at = off[None, :].expand_as(pg)
    s["weights_out"][pg[ok], :, at[ok]] = new[ok]
    return {"out": out, "weights": s["weights_out"]}


def _append(s):
    c = s["case"]
    rows = torch.arange(s["new_k"].shape[0], device=s["cu"].device)
    b = torch.searchsorted(s["cu"][1:].long(), rows, right=True)
    slot = s["starts"].long()[b] + rows - s["cu"].long()[b]
    pg = s["table"][b, slot // c["page"]].long()
    off = slot % c["page"]
    res = {}
    for name, new, bits in (("k", "new_k", BITS[c["kind"]][0]), ("v", "new_v", BITS[c["kind"]][1])):
        pool = s[name]
        if bits == 16:
            pool["x"][pg, :, off] = s[new]
            res[name] = pool["x"]
            continue
        for key, val in zip("xsb", _affine(s[new].float(), bits)):
            pool[key][pg, :, off] = val
        res[name] = [pool["x"], pool["s"], pool["b"]]
    return res


def _evict(s):
    c = s["case"]
    n, budget, hkv, page = max(1, c["hi"]), c["budget"], c["hkv"], c["page"]
    pg, off, idx = _slots(s, n)
    L = s["lengths"].long()
    w = s["weights"][pg, :, off].permute(0, 2, 1)  # [B, hkv, n]
    pos = s["positions"][pg, :, off].permute(0, 2, 1)
    there = (idx[None, :] < L[:, None])[:, None, :]
    kept_first = pos >= s["keep_from"].long()[:, None, None]
    key = torch.where(kept_first, torch.full_like(w, float("inf")), w)
    key = torch.where(there, key, torch.full_like(w, float("-inf")))
    rank = torch.sort(key, dim=-1, descending=True, stable=True).indices
    keep = torch.zeros_like(key, dtype=torch.bool)
    keep.scatter_(-1, rank[..., :budget], True)
    keep &= there
    hole = (idx < budget) & there & ~keep
    high = (idx >= budget) & keep
    # the r-th hole takes the r-th surviving row above the budget
    b, h, dst = torch.nonzero(hole, as_tuple=True)
    _, _, src = torch.nonzero(high, as_tuple=True)
    to = (pg[b, dst], h, dst % page)
    frm = (pg[b, src], h, src % page)
    for pool in (s["k"], s["v"]):
        for t in pool.values():
            t[to] = t[frm]
    stay = (idx < budget)[None, :] & (idx[None, :] < L[:, None])
    at = off[None, :].expand_as(pg)
    for a, o in (("weights", "weights_out"), ("positions", "positions_out")):
        s[o][pg[stay], :, at[stay]] = s[a][pg[stay], :, at[stay]]
        s[o][to] = s[a][frm]
    s["lengths_out"].copy_(s["lengths"].clamp_max(budget))
    return {"k": [t for _, t in sorted(s["k"].items())], "v": [t for _, t in sorted(s["v"].items())],
            "weights": s["weights_out"], "positions": s["positions_out"], "lengths": s["lengths_out"]}


def _logits(s):
    x = s["logits"].float()
    B, V = x.shape
    idx = torch.arange(s["history"].shape[1], device=x.device)
    h = s["history"].long()
    there = idx[None, :] < s["history_len"][:, None]
    said = there & (idx[None, :] >= s["prompt_len"][:, None])
    seen = torch.zeros(B, V, device=x.device).scatter_add_(1, h, there.float()) > 0
    count = torch.zeros(B, V, device=x.device).scatter_add_(1, h, said.float())
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x < 0, x * rep, x / rep), x)
    x = x - s["frequency"][:, None] * count
    x = torch.where(count > 0, x - s["presence"][:, None], x)
    if s["bias_ids"] is not None:
        m = s["bias_ids"].shape[1]
        last = torch.full((B, V + 1), -1, dtype=torch.long, device=x.device)
        ids = torch.where(s["bias_ids"] < 0, V, s["bias_ids"]).long()
        last.scatter_reduce_(1, ids, torch.arange(m, device=x.device)[None, :].expand(B, m), "amax")
        last = last[:, :V]
        x = torch.where(last >= 0, x + s["bias_values"].gather(1, last.clamp_min(0)), x)
    if s["allow"] is not None:
        i = torch.arange(V, device=x.device)
        x = torch.where(((s["allow"][:, i >> 5] >> (i & 31)) & 1).bool(), x, torch.full_like(x, float("-inf")))
    return {"logits": x.to(s["logits"].dtype)}


def _own(s):
    from rec_b200 import paged, sampling

    c = s["case"]
    if c["op"] == "logits":
        return {"logits": sampling.process_logits(
            s["logits"], history=s["history"], history_len=s["history_len"], prompt_len=s["prompt_len"],
            repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"], bias_ids=s["bias_ids"],
            bias_values=s["bias_values"], allow=s["allow"], out=s["out"])}
    k, v = s["k"], s["v"]
    cache = paged.PagedKV(k["x"], v["x"], k.get("s"), k.get("b"), v.get("s"), v.get("b"))
    if c["op"] == "append":
        paged.paged_append(cache, s["new_k"], s["new_v"], s["table"], s["starts"], s["cu"])
        return {n: p["x"] if "s" not in p else [p["x"], p["s"], p["b"]] for n, p in (("k", k), ("v", v))}
    if c["op"] == "attn":
        out = paged.paged_attn_decode(cache, s["q"], s["table"], s["lengths"], softcap=c["cap"], window=c["window"],
                                      sinks=s["sinks"], weights=s.get("weights"), weights_out=s.get("weights_out"),
                                      decay=0.98)
        return {"out": out, "weights": s["weights_out"]} if c["weights"] else {"out": out}
    paged.paged_evict(cache, s["table"], s["lengths"], c["budget"], s["weights"], positions=s["positions"],
                      keep_from=s["keep_from"], weights_out=s["weights_out"], positions_out=s["positions_out"],
                      lengths_out=s["lengths_out"])
    return {"k": [t for _, t in sorted(k.items())], "v": [t for _, t in sorted(v.items())],
            "weights": s["weights_out"], "positions": s["positions_out"], "lengths": s["lengths_out"]}


def run(state):
    if own:
        return _own(state)
    return {"attn": _attn, "append": _append, "evict": _evict, "logits": _logits}[state["case"]["op"]](state)


# --------------------------------------------------------------------------
# the definitions in 64 bits, one session (and kv head) at a time


def _exact_attn(s):
    c = s["case"]
    page, hkv, d = c["page"], c["hkv"], c["d"]
    kb, vb = BITS[c["kind"]]
    G = c["hq"] // hkv
    out = torch.zeros(c["batch"], c["hq"], d, dtype=torch.float64, device="cuda")
    acc = torch.zeros(s["weights"].shape, dtype=torch.float64, device="cuda") if c["weights"] else None
    for b, n in enumerate(s["lengths"].tolist()):
        if not n:
            continue
        t = torch.arange(n, device="cuda")
        where = s["table"][b, t // page].long()
        first = max(0, n - c["window"]) if c["window"] else 0
        for h in range(hkv):
            K = _values(s["k"], kb, lambda p: p[where[first:], h, t[first:] % page], torch.float64)
            V = _values(s["v"], vb, lambda p: p[where[first:], h, t[first:] % page], torch.float64)
            x = (s["q"][b, h * G:(h + 1) * G].double() @ K.T) / math.sqrt(d)
            if c["cap"]:
                x = torch.tanh(x / c["cap"]) * c["cap"]
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][h * G:(h + 1) * G].double()[:, None]], 1)
            p = torch.softmax(x, 1)[:, :n - first]
            out[b, h * G:(h + 1) * G] = p @ V
            if acc is not None:
                w = s["weights"][where, h, t % page].double() * 0.98
                w[first:] += p.sum(0)
                acc[where, h, t % page] = w
    return {"out": out, "weights": acc} if acc is not None else {"out": out}


def _exact_append(s):
    c = s["case"]
    res = {}
    starts, cu = s["starts"].tolist(), s["cu"].tolist()
    for name, bits in zip("kv", BITS[c["kind"]]):
        new = s["new_" + name].double()
        if bits == 16:
            parts = [new]
        else:
            w = new.reshape(*new.shape[:-1], -1, GROUP)
            hi, lo = w.max(-1).values, w.min(-1).values
            neg = lo.abs() > hi.abs()
            edge = torch.where(neg, lo, hi)
            step = torch.clamp((hi - lo) / (2 ** bits - 1), min=1e-7) * torch.where(neg, 1.0, -1.0)
            k = torch.round(edge / step)
            parts = [None, torch.where(k != 0, edge / k, step), torch.where(k != 0, edge, 0.0 * edge)]
        pools = []
        for key, val in zip("xsb", parts):
            if val is None:
                pools.append(None)
                continue
            pool = torch.zeros(s[name][key].shape, dtype=torch.float64, device="cuda")
            for b in range(c["batch"]):
                t = starts[b] + torch.arange(cu[b + 1] - cu[b], device="cuda")
                pool[s["table"][b, t // c["page"]].long(), :, t % c["page"]] = val[cu[b]:cu[b + 1]]
            pools.append(pool)
        res[name] = pools[0] if bits == 16 else pools
    return res


def _exact_logits(s):
    x = s["logits"].double()
    B, V = x.shape
    for b in range(B):
        n, m = int(s["history_len"][b]), int(s["prompt_len"][b])
        ids = s["history"][b, :n].long()
        rho = float(s["repetition"][b])
        u = torch.unique(ids)
        x[b, u] = torch.where(x[b, u] < 0, x[b, u] * rho, x[b, u] / rho)
        count = torch.bincount(ids[m:], minlength=V).double()
        x[b] -= float(s["frequency"][b]) * count + float(s["presence"][b]) * (count > 0)
        if s["bias_ids"] is not None:
            bias = dict((i, v) for i, v in zip(s["bias_ids"][b].tolist(), s["bias_values"][b].tolist()) if i >= 0)
            if bias:
                x[b, torch.tensor(list(bias), device="cuda")] += torch.tensor(list(bias.values()), device="cuda",
                                                                              dtype=torch.float64)
        if s["allow"] is not None:
            bits = (s["allow"][b][:, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
            x[b, bits.reshape(-1)[:V] == 0] = float("-inf")
    return {"logits": x}


def exact(case, seed):
    if case["op"] == "evict":
        return None  # selection and copies: nothing is computed that has a value in 64 bits
    s = prepare(case, seed)
    return {"attn": _exact_attn, "append": _exact_append, "logits": _exact_logits}[case["op"]](s)
