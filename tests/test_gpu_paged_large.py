"""The batched-decode operators at the sizes where they choose other launches:
long shares per SM, caches whose eviction keys leave shared memory, many moves,
many appended rows.  Float64 forms on the device, moves and rows by index.

Tolerances as for the small sizes: the attention's output is rounded once to
bf16 (relative 2^-8 at most per value, which the 2-norm of the difference is
held to); weights 2e-5 in the 2-norm.  Everything that is moved is equal bit
for bit."""
import numpy as np
import pytest
import torch

from rec_b200 import paged, sampling
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


def device_rows(pool, table, b, n, h):
    page = pool.shape[2]
    t = torch.arange(n, device="cuda")
    return pool[table[b, t // page].long(), h, t % page].double()


def norm_error(a, b):
    return float(torch.linalg.norm(a - b) / torch.linalg.norm(b))


@pytest.mark.parametrize("heads,group,lengths,window", [(1, 4, [300000, 5, 260001, 0, 3], 0), (2, 12, [131000, 200003], 0),
                                                        (1, 8, [400000, 350017], 300001)])
def test_attention_long_shares(heads, group, lengths, window):
    rng = np.random.default_rng(len(lengths))
    table, pages = ref.page_table(lengths, 128, rng)
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(pages, heads, 128, 64, device="cuda", generator=g).bfloat16() for _ in range(2))
    w = torch.rand(pages, heads, 128, device="cuda", generator=g)
    before = w.clone()
    q = (2 * torch.randn(len(lengths), heads * group, 64, device="cuda", generator=g)).bfloat16()
    t = torch.from_numpy(table).cuda()
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    cache = paged.PagedKV(k, v)
    out = paged.paged_attn_decode(cache, q, t, n, window=window)
    same = paged.paged_attn_decode(cache, q, t, n, window=window, weights=w, decay=0.5)
    paged.check_status()
    assert torch.equal(out, same)
    for b, L in enumerate(lengths):
        if L == 0:
            assert not bool(out[b].any())
            continue
        first = max(0, L - window) if window else 0
        slots = torch.arange(L, device="cuda")
        at = t[b, slots // 128].long()
        for h in range(heads):
            K, V = device_rows(k, t, b, L, h)[first:], device_rows(v, t, b, L, h)[first:]
            mine = slice(h * group, (h + 1) * group)
            p = torch.softmax(q[b, mine].double() @ K.T * 0.125, -1)
            assert norm_error(out[b, mine].double(), p @ V) <= 2.0 ** -8
            want = 0.5 * before[at, h, slots % 128].double()
            want[first:] += p.sum(0)
            assert norm_error(w[at, h, slots % 128].double(), want) <= 2e-5


def evict_by_sorting(w, prot, budget):
    """(holes, survivors) of one session and head."""
    nan = np.isnan(w)
    key = np.where(nan, 0.0, -w.astype(np.float64))
    n = len(w)
    order = np.lexsort((np.arange(n), np.where(prot, 0.0, key), np.where(prot, False, nan), ~prot))
    keep = np.zeros(n, dtype=bool)
    keep[order[:budget]] = True
    return np.flatnonzero(~keep[:budget]), budget + np.flatnonzero(keep[budget:])


@pytest.mark.parametrize("kb,vb,heads,d,page,lengths,budget", [
    (16, 16, 1, 8, 1000, [340000, 7, 327681], 170000),  # keys beyond shared memory
    (8, 4, 1, 64, 256, [330000], 329990),               # the same, few moves
    (16, 16, 4, 64, 64, [12000] * 8, 6000),             # many moves
    (4, 8, 4, 128, 64, [12000, 7000] * 4, 6000),
    (4, 4, 2, 256, 16, [9000] * 16, 4500)])
def test_evict_large(kb, vb, heads, d, page, lengths, budget):
    rng = np.random.default_rng(budget)
    table, pages = ref.page_table(lengths, page, rng)
    g = torch.Generator(device="cuda").manual_seed(4)
    cache = paged.PagedKV.allocate(pages, heads, page, d, k_bits=kb, v_bits=vb)
    pools = [x for x in (cache.k, cache.v, *cache.scales) if x is not None]
    for x in pools:
        bits = x.view(torch.int16)
        bits.copy_(torch.randint(-2 ** 15, 2 ** 15, bits.shape, device="cuda", generator=g, dtype=torch.int16))
    w = torch.rand(pages, heads, page, device="cuda", generator=g)
    w[torch.rand(w.shape, device="cuda", generator=g) < 0.4] = 0.25  # ties
    w[torch.rand(w.shape, device="cuda", generator=g) < 0.01] = float("nan")
    pos = torch.randint(0, 10 ** 6, w.shape, device="cuda", generator=g, dtype=torch.int32)
    t = torch.from_numpy(table).cuda()
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    keep_from = torch.full_like(n, 999_000)
    everything = [*pools, w, pos]
    want = [x.clone() for x in everything]
    w_host, pos_host = w.cpu().numpy(), pos.cpu().numpy()
    for b, L in enumerate(lengths):
        if L <= budget:
            continue
        pg, off = ref.rows_of(table, b, L, page)
        for h in range(heads):
            p = pos_host[pg, h, off]
            to, of = evict_by_sorting(w_host[pg, h, off], (p >= 999_000) | (p < 50), budget)
            assert len(to) == len(of) > 0
            at = [torch.from_numpy(i).cuda() for i in (pg[to], off[to], pg[of], off[of])]
            for x, y in zip(want, everything):
                x[at[0], h, at[1]] = y[at[2], h, at[3]]
    got = paged.paged_evict(cache, t, n, budget, w, positions=pos, keep_from=keep_from, keep_below=50, lengths_out=n)
    paged.check_status()
    assert got is n and n.tolist() == [min(L, budget) for L in lengths]  # the lengths in place
    for x, y in zip(want, everything):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


@pytest.mark.parametrize("kind,bits,heads,d", [("bf16", 16, 2, 64), ("fp16", 16, 5, 24), ("codes", 8, 3, 64),
                                               ("codes", 4, 1, 256)])
def test_append_many_rows(kind, bits, heads, d):
    """More rows than the small launch takes, and a last block that is not full."""
    rng = np.random.default_rng(d)
    counts = np.array([2000, 0, 1, 3000, 14])
    starts, page = np.array([5, 0, 100, 33, 16], dtype=np.int32), 48
    table, pages = ref.page_table(counts + starts, page, rng)
    dt = torch.float16 if kind == "fp16" else torch.bfloat16
    cache = paged.PagedKV.allocate(pages, heads, page, d, k_bits=bits, v_bits=bits, dtype=dt)
    pools = [x for x in (cache.k, cache.v, *cache.scales) if x is not None]
    for x in pools:
        x.zero_()
    total = int(counts.sum())
    x = rng.standard_normal((2, total, heads, d)).astype(np.float32)
    k, v = torch.from_numpy(x).cuda().to(dt)
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    w = torch.full((pages, heads, page), 7.0, device="cuda")
    pos = torch.full((pages, heads, page), -1, device="cuda", dtype=torch.int32)
    paged.paged_append(cache, k, v, torch.from_numpy(table).cuda(), torch.from_numpy(starts).cuda(),
                       torch.from_numpy(cu).cuda(), weights=w, positions=pos)
    paged.check_status()
    session = np.repeat(np.arange(len(counts)), counts)
    slot = starts[session] + np.arange(total) - cu[session]
    pg, off = (torch.from_numpy(i).cuda() for i in (table[session, slot // page].astype(np.int64), slot % page))
    for new, pool, (s, b) in ((k, cache.k, cache.scales[:2]), (v, cache.v, cache.scales[2:])):
        if bits == 16:
            parts = [(pool, new)]
        else:
            codes, es, eb = ref.affine(new.float().cpu().numpy(), bits)
            parts = [(pool, ref.pack(codes, bits).cuda()), (s, es.cuda()), (b, eb.cuda())]
        for have, rows in parts:
            want = torch.zeros_like(have)
            want[pg, :, off] = rows
            assert torch.equal(have, want)
    want = torch.full_like(pos, -1)
    want[pg, :, off] = torch.from_numpy(slot.astype(np.int32)).cuda()[:, None].expand(-1, heads)
    assert torch.equal(pos, want) and torch.equal(w, torch.where(want >= 0, 0.0, 7.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,V,n,m", [(70, 100_003, 5000, 40), (700, 9_300, 300, 3), (40, 151_936, 9000, 2000)])
def test_logit_rules_many_rows(dtype, B, V, n, m):
    """A batch of more than one wave equals its rows one at a time, bit for bit
    (those are held against the fp32 steps elsewhere)."""
    g = torch.Generator(device="cuda").manual_seed(V)
    i32 = dict(device="cuda", dtype=torch.int32)
    x = (4 * torch.randn(B, V, device="cuda", generator=g)).to(dtype)
    history = (torch.rand(B, n, device="cuda", generator=g) ** 3 * (V + 5)).int() - 2  # many repeats, some ids outside
    used = torch.randint(0, n + 1, (B,), generator=g, **i32)
    prompt = (used * torch.rand(B, device="cuda", generator=g)).int()
    numbers = [lo + torch.rand(B, device="cuda", generator=g) for lo in (1.0, 0.0, 0.0)]
    ids = (torch.rand(B, m, device="cuda", generator=g) ** 3 * V).int()
    ids[:, ::7] = -1
    ids[:, m // 2:] = history[:, :m - m // 2]
    values = torch.randn(B, m, device="cuda", generator=g)
    allow = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), device="cuda", generator=g).int()
    args = (history, used, prompt, *numbers, ids, values, allow)
    got = sampling.process_logits(x, *args)
    for b in range(0, B, 9):
        want = sampling.process_logits(x[b:b + 1], *(t[b:b + 1] for t in args))
        assert torch.equal(got[b], want[0])
    assert torch.equal(sampling.process_logits(x, *args, out=x), got)
