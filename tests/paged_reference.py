"""Plain float64 forms of the batched-decode operators (numpy, one session and
kv head at a time), and the inputs the tests share."""
import numpy as np
import torch


def affine(x: np.ndarray, bits: int):
    """MLX affine group-64 quantisation in fp32 steps: codes, bf16-rounded
    scale and bias (float64 values).  x float32 [..., D]."""
    f = np.float32
    w = x.astype(f).reshape(*x.shape[:-1], -1, 64)
    top, low = w.max(-1, keepdims=True), w.min(-1, keepdims=True)
    bins = f((1 << bits) - 1)
    step = np.maximum((top - low) / bins, f(1e-7))
    side = np.abs(low) > np.abs(top)
    step = np.where(side, step, -step).astype(f)
    edge = np.where(side, low, top).astype(f)
    q0 = np.rint(edge / step)
    scale = np.where(q0 != 0, edge / np.where(q0 != 0, q0, 1), step).astype(f)
    bias = np.where(q0 != 0, edge, 0).astype(f)
    codes = np.clip(np.rint((w - bias) / scale), 0, int(bins)).astype(np.int64)
    to_bf = lambda a: torch.from_numpy(np.ascontiguousarray(a[..., 0])).to(torch.bfloat16)  # noqa: E731
    return codes.reshape(x.shape), to_bf(scale), to_bf(bias)


def pack(codes: np.ndarray, bits: int) -> torch.Tensor:
    per = 32 // bits
    c = codes.reshape(*codes.shape[:-1], -1, per).astype(np.uint64)
    words = (c << (np.arange(per, dtype=np.uint64) * bits)).sum(-1).astype(np.uint32)
    return torch.from_numpy(words.view(np.int32))


def unpack(words: torch.Tensor, bits: int) -> np.ndarray:
    w = words.cpu().numpy().view(np.uint32)
    per = 32 // bits
    c = (w[..., None] >> (np.arange(per, dtype=np.uint32) * bits)) & ((1 << bits) - 1)
    return c.reshape(*w.shape[:-1], -1)


def values(x: torch.Tensor, bits: int, s=None, b=None) -> np.ndarray:
    """float64 values of a pool."""
    if bits == 16:
        return x.double().cpu().numpy()
    c = unpack(x, bits).astype(np.float64)
    c = c.reshape(*c.shape[:-1], -1, 64)
    c = c * s.double().cpu().numpy()[..., None] + b.double().cpu().numpy()[..., None]
    return c.reshape(*c.shape[:-2], -1)


def rows_of(table, b, n, page):
    t = np.arange(n)
    return np.asarray(table)[b, t // page].astype(np.int64), t % page


def attention(q, K, V, table, lengths, page, scale, cap=0.0, window=0, sinks=None, weights=None, decay=1.0):
    """(out, lse, weights_out) in float64; K, V float64 pools
    [pages, heads, page, D]; rows that a page id < 0 holds are left out."""
    B, hq, d = q.shape
    H = K.shape[1]
    G = hq // H
    out = np.zeros((B, hq, d))
    lse = np.full((B, hq), -np.inf)
    w_out = None if weights is None else weights.copy()
    for b in range(B):
        n = int(lengths[b])
        pg, off = rows_of(table, b, n, page)
        first = max(0, n - window) if window else 0
        seen = (np.arange(n) >= first) & (pg >= 0) & (pg < K.shape[0])
        for h in range(H):
            total = np.zeros(n)
            for g in range(h * G, (h + 1) * G):
                x = q[b, g] @ K[pg[seen], h, off[seen]].T * scale
                if cap:
                    x = cap * np.tanh(x / cap)
                ref = list(x) + ([sinks[g]] if sinks is not None else [])
                if not ref:
                    continue
                m = max(ref)
                den = sum(np.exp(np.asarray(ref) - m))
                p = np.exp(x - m) / den
                out[b, g] = p @ V[pg[seen], h, off[seen]]
                lse[b, g] = m + np.log(den)
                total[seen] += p
            if w_out is not None:
                ok = (pg >= 0) & (pg < K.shape[0])
                old = w_out[pg[ok], h, off[ok]]
                w_out[pg[ok], h, off[ok]] = (decay * old if decay else 0.0) + total[ok]
    return out, lse, w_out


def evict_plan(weights, positions, n, budget, keep_from, keep_below):
    """(kept slots below the budget stay) -> list of (hole, survivor)."""
    w = np.asarray(weights, dtype=np.float64)
    prot = (positions >= keep_from) | (positions < keep_below)
    order = sorted(range(n), key=lambda t: (not prot[t], np.isnan(w[t]), -w[t] if not np.isnan(w[t]) else 0.0, t)
                   if not prot[t] else (False, False, 0.0, t))
    keep = set(order[:budget])
    holes = [t for t in range(min(n, budget)) if t not in keep]
    highs = [t for t in range(budget, n) if t in keep]
    assert len(holes) == len(highs)
    return list(zip(holes, highs))


def logit_rules(x, history, prompt, rep, freq, pres, bias, allowed, dt=np.float64):
    """One row, every step in `dt`.  history: ids in use; bias: [(id, value)];
    allowed: bool [V] or None."""
    x = x.astype(dt)
    V = x.shape[0]
    rep, freq, pres = dt(rep), dt(freq), dt(pres)
    ok = lambda ids: [i for i in ids if 0 <= i < V]  # noqa: E731
    for i in set(ok(history)):
        x[i] = x[i] * rep if x[i] < 0 else x[i] / rep
    count = np.bincount(np.asarray(ok(history[prompt:]), dtype=np.int64), minlength=V).astype(dt)
    x = np.where(count > 0, x - freq * count - pres, x)
    for i, v in dict((i, v) for i, v in bias if 0 <= i < V).items():
        x[i] += dt(v)
    if allowed is not None:
        x = np.where(allowed, x, dt(-np.inf))
    return x


def page_table(lengths, page, rng, spare=2, width=None):
    """A shuffled page table (unused entries -1) and the page count."""
    need = [-(-int(n) // page) for n in lengths]
    total = sum(need) + spare
    order = rng.permutation(total)
    width = max(1, max(need)) if width is None else width
    table = np.full((len(need), width), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def quantized_pool(rng, pages, heads, page, d, bits, device):
    x = rng.standard_normal((pages, heads, page, d)).astype(np.float32)
    codes, s, b = affine(x, bits)
    return pack(codes, bits).to(device), s.to(device), b.to(device)
