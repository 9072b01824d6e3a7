"""Batched decode over a paged cache on the GPU against float64 forms:
append, attention of one new token per session, eviction.

Tolerances.  Attention: the output is rounded once to its 16-bit type, a
relative error of at most 2^-8 (bf16) or 2^-11 (fp16) per value, and that is
what the 2-norm of the difference is held to (a rounding alone gives about a
third of it).  A score is a sum of D products in fp32: it is off by at most
D 2^-23 scale sum|q k|, which for these inputs (|q| about 2, |k| about 1)
stays below e = 2^-10; a weight is then off by at most 2 e relatively, and a
single output by 4 e max|v| in the worst case of all errors aligned.  Weights
and lse are fp32: 2e-5 in the 2-norm."""
import numpy as np
import pytest
import torch

from rec_b200 import paged
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

KINDS = {"bf16": (16, 16), "fp16": (16, 16), "k8v8": (8, 8), "k4v4": (4, 4), "k8v4": (8, 4), "k4v8": (4, 8)}


def make_cache(rng, kind, pages, heads, page, d):
    kb, vb = KINDS[kind]
    if kb == 16:
        dt = torch.float16 if kind == "fp16" else torch.bfloat16
        k, v = (torch.from_numpy(rng.standard_normal((pages, heads, page, d)).astype(np.float32)).cuda().to(dt)
                for _ in range(2))
        return paged.PagedKV(k, v), ref.values(k, 16), ref.values(v, 16)
    k = ref.quantized_pool(rng, pages, heads, page, d, kb, "cuda")
    v = ref.quantized_pool(rng, pages, heads, page, d, vb, "cuda")
    cache = paged.PagedKV(k[0], v[0], k[1], k[2], v[1], v[2])
    return cache, ref.values(k[0], kb, *k[1:]), ref.values(v[0], vb, *v[1:])


def rel(a, b):
    n = np.linalg.norm(b)
    return np.linalg.norm(a - b) / n if n else np.abs(a).max(initial=0.0)


def check_attention(kind, hq, heads, d, page, lengths, *, cap=0.0, window=0, sinks=False, weights=False, decay=1.0,
                    seed=0, scale=None):
    rng = np.random.default_rng(seed)
    lengths = np.asarray(lengths, dtype=np.int32)
    table, pages = ref.page_table(lengths, page, rng)
    cache, K, V = make_cache(rng, kind, pages, heads, page, d)
    dt = cache.dtype
    q = torch.from_numpy(2 * rng.standard_normal((len(lengths), hq, d)).astype(np.float32)).cuda().to(dt)
    sk = torch.from_numpy(rng.standard_normal(hq).astype(np.float32)).cuda().to(torch.bfloat16) if sinks else None
    w = torch.from_numpy(rng.random((pages, heads, page)).astype(np.float32)).cuda() if weights else None
    w0 = None if w is None else w.double().cpu().numpy()
    lse = torch.empty(len(lengths), hq, device="cuda")
    out = paged.paged_attn_decode(cache, q, torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda(),
                                  softcap=cap, window=window, sinks=sk, lse=lse, weights=w, decay=decay, scale=scale)
    paged.check_status()
    eo, el, ew = ref.attention(q.double().cpu().numpy(), K, V, table, lengths, page,
                               d ** -0.5 if scale is None else scale, cap, window,
                               None if sk is None else sk.double().cpu().numpy(), w0, decay)
    u = 2.0 ** -9 if dt == torch.bfloat16 else 2.0 ** -12
    o = out.double().cpu().numpy()
    assert np.isfinite(o).all()
    assert rel(o, eo) <= 2 * u
    assert np.abs(o - eo).max(initial=0) <= u * np.abs(eo).max(initial=0) + 4 * 2.0 ** -10 * np.abs(V).max()
    got = lse.double().cpu().numpy()
    inf = np.isinf(el)
    assert (got[inf] == -np.inf).all() and np.abs(got[~inf] - el[~inf]).max(initial=0) <= 2e-4
    assert rel(got[~inf], el[~inf]) <= 2e-5
    if weights:
        assert rel(w.double().cpu().numpy(), ew) <= 2e-5


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 5, 8, 13])
def test_attention_formats(kind, d, group):
    check_attention(kind, 2 * group, 2, d, 16, [0, 1, 7, 16, 17, 300, 1025], seed=d + group)


@pytest.mark.parametrize("d", [8, 24, 80, 96, 192, 248])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_attention_other_head_dims(kind, d):
    check_attention(kind, 12, 3, d, 24, [33, 0, 500], seed=d, sinks=True)


@pytest.mark.parametrize("page", [1, 3, 16, 48, 256, 1000])
@pytest.mark.parametrize("kind", ["bf16", "k8v4"])
def test_attention_pages(kind, page):
    check_attention(kind, 8, 1, 128, page, [1, 255, 256, 257, 2049], seed=page)


@pytest.mark.parametrize("kind", ["bf16", "k8v8", "k4v4"])
@pytest.mark.parametrize("window,cap,sinks", [(1, 0.0, False), (100, 30.0, True), (513, 0.0, True), (10 ** 6, 5.0, False)])
def test_attention_window_cap_sinks(kind, window, cap, sinks):
    check_attention(kind, 10, 2, 128, 32, [0, 1, 99, 100, 101, 700, 3000], window=window, cap=cap, sinks=sinks)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("decay", [0.0, 0.5, 1.0])
def test_attention_weights(kind, decay):
    check_attention(kind, 12, 2, 128, 16, [0, 1, 50, 777, 2000], weights=True, decay=decay, window=600, sinks=True)


@pytest.mark.parametrize("group", [1, 3, 16, 33])
def test_attention_weights_groups(group):
    check_attention("bf16", 2 * group, 2, 64, 64, [129, 1, 0, 1000], weights=True)


@pytest.mark.parametrize("kind", ["bf16", "k8v8", "k4v4"])
def test_attention_long(kind):
    """Few rows over a long cache: split over the length and joined."""
    check_attention(kind, 8, 1, 128, 256, [40000], seed=3)


def test_attention_many_sessions():
    rng = np.random.default_rng(5)
    check_attention("bf16", 4, 2, 64, 16, rng.integers(0, 40, 700), seed=5)
    check_attention("k8v8", 8, 1, 64, 16, rng.integers(0, 300, 200), seed=6)


def test_attention_dominant_and_far_scores():
    """A slot whose score is far above the others' (late in the cache), and
    scores that all lie far below zero."""
    for sign in (1.0, -1.0):
        rng = np.random.default_rng(1)
        table, pages = ref.page_table([900], 16, rng)
        k = torch.from_numpy(0.01 * rng.standard_normal((pages, 1, 16, 128)).astype(np.float32)).cuda().bfloat16()
        v = torch.from_numpy(rng.standard_normal((pages, 1, 16, 128)).astype(np.float32)).cuda().bfloat16()
        q = torch.ones(1, 8, 128, device="cuda", dtype=torch.bfloat16)
        k[table[0, 50], 0, 3] = 4.0 * sign if sign > 0 else -4.0
        if sign < 0:
            k -= 20.0
        out = paged.paged_attn_decode(paged.PagedKV(k, v), q, torch.from_numpy(table).cuda(),
                                      torch.tensor([900], device="cuda", dtype=torch.int32))
        eo, _, _ = ref.attention(q.double().cpu().numpy(), ref.values(k, 16), ref.values(v, 16), table, [900], 16,
                                 128 ** -0.5)
        assert rel(out.double().cpu().numpy(), eo) <= 2 * 2.0 ** -9


@pytest.mark.parametrize("kind", ["bf16", "fp16", "k8v8"])
def test_attention_ignores_what_is_masked(kind):
    """NaN and infinities in slots past the length, below the window and in
    pages of nobody change nothing."""
    rng = np.random.default_rng(2)
    lengths = np.array([70, 5, 0, 200], dtype=np.int32)
    page, window = 16, 60
    table, pages = ref.page_table(lengths, page, rng)
    cache, K, V = make_cache(rng, kind, pages, 2, page, 128)
    q = torch.from_numpy(rng.standard_normal((4, 16, 128)).astype(np.float32)).cuda().to(cache.dtype)
    t, n = torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda()
    clean = paged.paged_attn_decode(cache, q, t, n, window=window)
    seen = np.zeros((pages, page), dtype=bool)
    for b, L in enumerate(lengths):
        pg, off = ref.rows_of(table, b, L, page)
        first = max(0, L - window)
        seen[pg[first:], off[first:]] = True
    dead = torch.from_numpy(~seen).cuda()
    for x in (cache.k, cache.v, *cache.scales):
        if x is not None and x.dtype != torch.int32:
            x.permute(0, 2, 1, 3)[dead] = float("nan")
            x.permute(0, 2, 1, 3)[:, 1::2][dead[:, 1::2]] = float("inf")
    again = paged.paged_attn_decode(cache, q, t, n, window=window)
    assert torch.equal(clean, again)
    paged.check_status()


def test_attention_low_scores_and_empty_rows():
    """Keys at the type's lowest value, and sessions without a slot."""
    k = torch.full((2, 1, 16, 64), torch.finfo(torch.bfloat16).min, device="cuda", dtype=torch.bfloat16)
    v = torch.ones(2, 1, 16, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(2, 3, 64, device="cuda", dtype=torch.bfloat16)
    q[0, :, 0] = 1e-3
    t = torch.tensor([[0], [1]], device="cuda", dtype=torch.int32)
    lse = torch.zeros(2, 3, device="cuda")
    out = paged.paged_attn_decode(paged.PagedKV(k, v), q, t, torch.tensor([9, 0], device="cuda", dtype=torch.int32), lse=lse)
    assert torch.equal(out[0], torch.ones_like(out[0])) and torch.equal(out[1], torch.zeros_like(out[1]))
    assert (lse[1] == float("-inf")).all()


def test_attention_repeats_bit_for_bit():
    rng = np.random.default_rng(8)
    lengths = np.array([5000, 3, 12000, 777], dtype=np.int32)
    table, pages = ref.page_table(lengths, 32, rng)
    cache, _, _ = make_cache(rng, "bf16", pages, 2, 32, 128)
    q = torch.randn(4, 16, 128, device="cuda").bfloat16()
    t, n = torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda()
    first = paged.paged_attn_decode(cache, q, t, n)
    for _ in range(20):
        assert torch.equal(paged.paged_attn_decode(cache, q, t, n), first)


def test_attention_layouts_and_strides():
    """Pools whose rows are not in the default order (slot before head, a
    slice of a wider pool) and q / out that are slices."""
    rng = np.random.default_rng(4)
    lengths = np.array([100, 37], dtype=np.int32)
    table, pages = ref.page_table(lengths, 16, rng)
    wide = torch.randn(pages, 16, 3, 2, 192, device="cuda").bfloat16()  # page, slot, head, k/v, dim
    k, v = (wide[:, :, :, i, 64:].permute(0, 2, 1, 3) for i in (0, 1))
    qkv = torch.randn(2, 9, 128, device="cuda").bfloat16()
    big = torch.zeros(2, 12, 128, device="cuda").bfloat16()
    t = torch.from_numpy(np.concatenate([table, table], 1)).cuda()[:, :table.shape[1]]
    out = paged.paged_attn_decode(paged.PagedKV(k, v), qkv[:, :6], t, torch.from_numpy(lengths).cuda(), out=big[:, 3:9])
    eo, _, _ = ref.attention(qkv[:, :6].double().cpu().numpy(), ref.values(k, 16), ref.values(v, 16), table, lengths, 16,
                             128 ** -0.5)
    assert out.data_ptr() == big[:, 3:9].data_ptr() and rel(out.double().cpu().numpy(), eo) <= 2 * 2.0 ** -9
    assert not big[:, :3].any() and not big[:, 9:].any()


def test_attention_past_32_bit_offsets():
    """Pages more than 2^32 bytes and 2^31 elements into the pool."""
    pages, page = 5000, 256
    k = torch.empty(pages, 4, page, 128, device="cuda", dtype=torch.bfloat16)  # 1.3 GB
    big = torch.empty(4 * pages, 4, page, 128, device="cuda", dtype=torch.bfloat16)  # 5.2 GB
    ids = torch.tensor([[4 * pages - 1, 4 * pages - 7]], device="cuda", dtype=torch.int32)
    small = torch.randn(2, 4, page, 128, device="cuda").bfloat16()
    big[ids[0].long()] = small
    q = torch.randn(1, 8, 128, device="cuda").bfloat16()
    n = torch.tensor([400], device="cuda", dtype=torch.int32)
    got = paged.paged_attn_decode(paged.PagedKV(big, big), q, ids, n)
    want = paged.paged_attn_decode(paged.PagedKV(small, small), q, torch.tensor([[0, 1]], device="cuda", dtype=torch.int32), n)
    assert torch.equal(got, want)
    del k


def test_attention_other_stream_and_graph():
    rng = np.random.default_rng(9)
    lengths = np.array([900, 20], dtype=np.int32)
    table, pages = ref.page_table(lengths, 16, rng)
    cache, _, _ = make_cache(rng, "bf16", pages, 2, 16, 64)
    q = torch.randn(2, 8, 64, device="cuda").bfloat16()
    w = torch.zeros(*cache.shape, device="cuda")
    t, n = torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda()
    want = paged.paged_attn_decode(cache, q, t, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged.paged_attn_decode(cache, q, t, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.paged_attn_decode(cache, q, t, n, out=out, weights=w, decay=1.0)
    for i in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert abs(float(w.sum()) - 3 * 2 * 8) < 1e-2  # each head's weights sum to 1 per replay


def test_bad_pages_are_left_out_and_reported():
    rng = np.random.default_rng(10)
    lengths = np.array([64], dtype=np.int32)
    table, pages = ref.page_table(lengths, 16, rng)
    cache, K, V = make_cache(rng, "bf16", pages, 1, 16, 64)
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    for bad in (-1, pages, 2 ** 31 - 1):
        broken = table.copy()
        broken[0, 2] = bad
        out = paged.paged_attn_decode(cache, q, torch.from_numpy(broken).cuda(), torch.from_numpy(lengths).cuda())
        eo, _, _ = ref.attention(q.double().cpu().numpy(), K, V, broken, lengths, 16, 0.125)
        assert rel(out.double().cpu().numpy(), eo) <= 2 * 2.0 ** -9
        with pytest.raises(RuntimeError, match="status 5"):
            paged.check_status()
        paged.check_status()
    # a length past the table
    paged.paged_attn_decode(cache, q, torch.from_numpy(table).cuda(), torch.tensor([65], device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError, match="status 5"):
        paged.check_status()


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("d", [64, 128, 256])
def test_append(kind, d):
    rng = np.random.default_rng(d)
    kb, vb = KINDS[kind]
    counts, starts, page, heads = np.array([3, 0, 1, 40, 17]), np.array([0, 5, 31, 7, 16], dtype=np.int32), 16, 3
    table, pages = ref.page_table(counts + starts, page, rng)
    dt = torch.float16 if kind == "fp16" else torch.bfloat16
    cache = paged.PagedKV.allocate(pages, heads, page, d, k_bits=kb, v_bits=vb, dtype=dt)
    for x in (cache.k, cache.v, *cache.scales):
        if x is not None:
            x.zero_()
    total = int(counts.sum())
    wide = torch.from_numpy(rng.standard_normal((total, 2, heads, d)).astype(np.float32)).cuda().to(dt)
    k, v = wide[:, 0], wide[:, 1]
    k[0, 0, :64] = 0.0  # a group of equal values
    k[1, 1, :64] = 1.5
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    w = torch.full((pages, heads, page), 7.0, device="cuda")
    pos = torch.full((pages, heads, page), -1, device="cuda", dtype=torch.int32)
    paged.paged_append(cache, k, v, torch.from_numpy(table).cuda(), torch.from_numpy(starts).cuda(),
                       torch.from_numpy(cu).cuda(), weights=w, positions=pos)
    paged.check_status()
    for new, pool, bits, s, b in ((k, cache.k, kb, *cache.scales[:2]), (v, cache.v, vb, *cache.scales[2:])):
        x = new.float().cpu().numpy()
        if bits == 16:
            want = torch.zeros_like(pool)
        else:
            codes, es, eb = ref.affine(x, bits)
            want, want_s, want_b = torch.zeros_like(pool), torch.zeros_like(s), torch.zeros_like(b)
            words = ref.pack(codes, bits).cuda()
        for i, n in enumerate(counts):
            for j in range(n):
                slot, r = starts[i] + j, cu[i] + j
                pg, off = table[i, slot // page], slot % page
                if bits == 16:
                    want[pg, :, off] = new[r]
                else:
                    want[pg, :, off] = words[r]
                    want_s[pg, :, off], want_b[pg, :, off] = es[r].cuda(), eb[r].cuda()
                assert (pos[pg, :, off] == int(slot)).all() and (w[pg, :, off] == 0).all()
        assert torch.equal(pool, want)
        if bits != 16:
            assert torch.equal(s, want_s) and torch.equal(b, want_b)
    assert int((pos >= 0).sum()) == total * heads and int((w == 7).sum()) == w.numel() - total * heads


def test_append_equals_the_single_session_append():
    """The codes of rec_kv_append_bulk, row by row."""
    import ctypes as C

    from rec_b200 import abi
    from rec_b200._lib import check, lib

    heads, n, page = 2, 256, 64
    k, v = (torch.randn(n, heads, 128, device="cuda").bfloat16() for _ in range(2))
    # quotients that lie on and beside halves
    g = torch.Generator(device="cuda").manual_seed(1)
    k[::2] = (torch.randint(-255, 256, k[::2].shape, device="cuda", generator=g).float() / 2).bfloat16()
    v[::2] = (torch.randint(0, 511, v[::2].shape, device="cuda", generator=g).float() / 2).bfloat16()
    v[::2, :, ::64] = 255.0
    v[::2, :, 1::64] = 0.0
    flat = dict(k_codes=torch.zeros(heads, n, 32, dtype=torch.int32, device="cuda"))
    flat["v_codes"] = torch.zeros_like(flat["k_codes"])
    for name in ("k_scales", "k_biases", "v_scales", "v_biases"):
        flat[name] = torch.zeros(heads, n, 2, dtype=torch.bfloat16, device="cuda")
    layer = abi.RecKVLayer(**{a: t.data_ptr() for a, t in flat.items()})
    check(lib().rec_kv_append_bulk(C.byref(layer), heads, n, 8, k.data_ptr(), v.data_ptr(), 0, n,
                                   torch.cuda.current_stream().cuda_stream))
    cache = paged.PagedKV.allocate(n // page, heads, page, 128, k_bits=8, v_bits=8)
    table = torch.arange(n // page, device="cuda", dtype=torch.int32)[None]
    paged.paged_append(cache, k, v, table, torch.zeros(1, device="cuda", dtype=torch.int32),
                       torch.tensor([0, n], device="cuda", dtype=torch.int32))
    for got, want in ((cache.k, "k_codes"), (cache.v, "v_codes"), (cache.scales[0], "k_scales"),
                      (cache.scales[3], "v_biases")):
        assert torch.equal(got.permute(1, 0, 2, 3).reshape(heads, n, -1), flat[want])


def test_append_bad_slots_are_left_out_and_reported():
    cache = paged.PagedKV.allocate(2, 1, 16, 64)
    cache.k.zero_(), cache.v.zero_()
    k = torch.ones(4, 1, 64, device="cuda").bfloat16()
    table = torch.tensor([[0, 9], [1, -1]], device="cuda", dtype=torch.int32)
    i32 = dict(device="cuda", dtype=torch.int32)
    cu = torch.tensor([0, 2, 4], **i32)
    for starts, code, written in (([15, 0], 5, 3), ([31, 4], 5, 2), ([-1, 15], 4, 2)):
        cache.k.zero_()
        paged.paged_append(cache, k, k, table, torch.tensor(starts, **i32), cu)
        with pytest.raises(RuntimeError, match="status"):
            paged.check_status()
        assert int((cache.k[:, :, :, 0] != 0).sum()) == written
    # rows that cu_seqlens does not cover are not written
    cache.k.zero_()
    paged.paged_append(cache, k, k, table, torch.zeros(2, **i32), torch.tensor([0, 1, 2], **i32))
    paged.check_status()
    assert int((cache.k[:, :, :, 0] != 0).sum()) == 2


def check_evict(kind, lengths, budget, *, heads=2, page=16, d=128, recent=None, keep_below=0, in_place=True, seed=0,
                weights=None, positions=True):
    rng = np.random.default_rng(seed)
    lengths = np.asarray(lengths, dtype=np.int32)
    table, pages = ref.page_table(lengths, page, rng)
    cache, _, _ = make_cache(rng, kind, pages, heads, page, d)
    w = rng.random((pages, heads, page)).astype(np.float32) ** 4
    w[rng.random(w.shape) < 0.3] = 0.0
    if weights is not None:
        w = weights(rng, w)
    pos = np.full((pages, heads, page), -5, dtype=np.int32)
    for b, n in enumerate(lengths):
        pg, off = ref.rows_of(table, b, n, page)
        for h in range(heads):
            pos[pg, h, off] = rng.permutation(int(n)) if positions == "shuffled" else np.arange(n)
    keep_from = None if recent is None else (lengths - recent).astype(np.int32)
    names = [x for x in (cache.k, cache.v, *cache.scales) if x is not None]
    want = [x.cpu().clone() for x in names]
    ww, wp = w.copy(), pos.copy()
    for b, n in enumerate(lengths):
        pg, off = ref.rows_of(table, b, n, page)
        for h in range(heads):
            plan = ref.evict_plan(w[pg, h, off], pos[pg, h, off] if positions else np.arange(n), int(n), budget,
                                  2 ** 31 - 1 if keep_from is None else keep_from[b], keep_below)
            for dst, src in plan:
                for x in want:
                    x[pg[dst], h, off[dst]] = x[pg[src], h, off[src]]
                ww[pg[dst], h, off[dst]] = w[pg[src], h, off[src]]
                wp[pg[dst], h, off[dst]] = pos[pg[src], h, off[src]]
    cw, cp = torch.from_numpy(w).cuda(), torch.from_numpy(pos).cuda()
    t, n = torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda()
    kf = None if keep_from is None else torch.from_numpy(keep_from).cuda()
    outs = dict(weights_out=torch.full_like(cw, -1.0), positions_out=torch.full_like(cp, -9)) if not in_place else {}
    got = paged.paged_evict(cache, t, n, budget, cw, positions=cp if positions else None, keep_from=kf,
                            keep_below=keep_below, **outs)
    paged.check_status()
    assert got.cpu().tolist() == np.minimum(lengths, budget).tolist()
    for x, y in zip(names, want):
        assert torch.equal(x.cpu().view(torch.int16 if x.element_size() == 2 else torch.int32),
                           y.view(torch.int16 if y.element_size() == 2 else torch.int32))
    if in_place:
        assert np.array_equal(cw.cpu().numpy(), ww, equal_nan=True)
        if positions:
            assert np.array_equal(cp.cpu().numpy(), wp)
        return
    for b, L in enumerate(lengths):
        pg, off = ref.rows_of(table, b, min(int(L), budget), page)
        assert np.array_equal(outs["weights_out"].cpu().numpy()[pg, :, off], ww[pg, :, off], equal_nan=True)
        if positions:
            assert np.array_equal(outs["positions_out"].cpu().numpy()[pg, :, off], wp[pg, :, off])
    assert np.array_equal(cw.cpu().numpy(), w, equal_nan=True)  # the inputs stay


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_formats(kind, in_place):
    check_evict(kind, [0, 1, 40, 41, 300, 1111], 40, recent=8, in_place=in_place)


@pytest.mark.parametrize("budget", [0, 1, 63, 64, 65, 999, 1000, 1001, 5000])
def test_evict_budgets(budget):
    check_evict("bf16", [1000, 64, 2, 0], budget, d=64, page=24, seed=budget)


@pytest.mark.parametrize("recent,keep_below", [(None, 0), (0, 4), (30, 4), (200, 0), (70, 0)])
def test_evict_protected(recent, keep_below):
    """Protected slots first; more of them than the budget leaves the lowest."""
    check_evict("bf16", [500, 90], 70, recent=recent, keep_below=keep_below, positions="shuffled", d=64)


def test_evict_without_positions():
    check_evict("fp16", [500, 90], 70, recent=16, keep_below=2, positions=None, d=64)


@pytest.mark.parametrize("fill", ["equal", "zeros", "nan", "inf", "negative"])
def test_evict_ties_and_odd_weights(fill):
    def weights(rng, w):
        if fill == "equal":
            return np.full_like(w, 0.25)
        if fill == "zeros":
            return np.where(rng.random(w.shape) < 0.5, np.float32(0.0), np.float32(-0.0))
        if fill == "nan":
            return np.where(rng.random(w.shape) < 0.7, np.float32("nan"), w)
        if fill == "inf":
            return np.where(rng.random(w.shape) < 0.7, np.float32("inf"), np.float32("-inf"))
        return -w
    check_evict("bf16", [300, 77], 64, recent=10, weights=weights, d=64)


@pytest.mark.parametrize("lengths,budget", [([20000], 3000), ([9000, 12345], 9000), ([70000], 65536)])
def test_evict_long(lengths, budget):
    check_evict("k8v4", lengths, budget, heads=1, page=256, d=64, recent=100)


def test_append_attend_evict_as_a_session_runs_them():
    """Sessions that grow token by token under a budget: the cache, the
    weights and the positions stay those of a float64 run of the same steps."""
    rng = np.random.default_rng(12)
    B, heads, hq, d, page, budget, recent = 3, 2, 4, 64, 8, 24, 8
    table, pages = ref.page_table([budget + page] * B, page, rng)
    cache = paged.PagedKV.allocate(pages, heads, page, d)
    cache.k.zero_(), cache.v.zero_()
    w = torch.zeros(pages, heads, page, device="cuda")
    pos = torch.zeros(pages, heads, page, device="cuda", dtype=torch.int32)
    t = torch.from_numpy(table).cuda()
    n = torch.zeros(B, device="cuda", dtype=torch.int32)
    cu = torch.arange(B + 1, device="cuda", dtype=torch.int32)
    seen = [0] * B
    for step in range(60):
        k, v = (torch.from_numpy(rng.standard_normal((B, heads, d)).astype(np.float32)).cuda().bfloat16() for _ in range(2))
        q = torch.from_numpy(rng.standard_normal((B, hq, d)).astype(np.float32)).cuda().bfloat16()
        paged.paged_append(cache, k, v, t, n, cu, weights=w, positions=pos)
        n += 1
        lengths = n.cpu().numpy()
        for b in range(B):  # the position of the new slot is the token's own
            pg, off = ref.rows_of(table, b, lengths[b], page)
            pos[pg[-1], :, off[-1]] = step
        before = w.double().cpu().numpy()
        out = paged.paged_attn_decode(cache, q, t, n, weights=w)
        eo, _, ew = ref.attention(q.double().cpu().numpy(), ref.values(cache.k, 16), ref.values(cache.v, 16), table,
                                  lengths, page, d ** -0.5, weights=before)
        assert rel(out.double().cpu().numpy(), eo) <= 2 * 2.0 ** -9 and rel(w.double().cpu().numpy(), ew) <= 2e-5
        if lengths[0] == budget + page:
            n = paged.paged_evict(cache, t, n, budget, w, positions=pos,
                                  keep_from=torch.full((B,), step + 1 - recent, device="cuda", dtype=torch.int32))
            p = pos.cpu().numpy()
            for b in range(B):
                pg, off = ref.rows_of(table, b, budget, page)
                for h in range(heads):
                    have = p[pg, h, off]
                    assert len(set(have.tolist())) == budget and set(range(step + 1 - recent, step + 1)) <= set(have.tolist())
    paged.check_status()


def test_python_refusals():
    k = torch.zeros(4, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    i32 = dict(device="cuda", dtype=torch.int32)
    cache = paged.PagedKV(k, k.clone())
    t, n = torch.zeros(3, 2, **i32), torch.zeros(3, **i32)
    q = torch.zeros(3, 8, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(4, 2, 16, device="cuda")
    for bad in (lambda: paged.PagedKV(k, k[:3]), lambda: paged.PagedKV(k, k.half()), lambda: paged.PagedKV(k[0], k[0]),
                lambda: paged.PagedKV(k.float(), k.float()), lambda: paged.PagedKV(k.transpose(2, 3), k.transpose(2, 3)),
                lambda: paged.PagedKV(k, k, *[k[..., :1]] * 4),
                lambda: paged.PagedKV.allocate(2, 1, 16, 80, k_bits=8, v_bits=8),
                lambda: paged.paged_attn_decode(cache, q.half(), t, n), lambda: paged.paged_attn_decode(cache, q[:2], t, n),
                lambda: paged.paged_attn_decode(cache, q, t.long(), n), lambda: paged.paged_attn_decode(cache, q, t, n[:2]),
                lambda: paged.paged_attn_decode(cache, q, t, n.long()), lambda: paged.paged_attn_decode(cache, q[:, :7], t, n),
                lambda: paged.paged_attn_decode(cache, q, t, n, out=q.float()),
                lambda: paged.paged_attn_decode(cache, q, t, n, sinks=torch.zeros(8, device="cuda")),
                lambda: paged.paged_attn_decode(cache, q, t, n, weights=w[:2]),
                lambda: paged.paged_attn_decode(cache, q, t, n, window=-1),
                lambda: paged.paged_attn_decode(cache, q.cpu(), t, n),
                lambda: paged.paged_evict(cache, t, n, -1, w), lambda: paged.paged_evict(cache, t, n, 4, w.half()),
                lambda: paged.paged_evict(cache, t, n, 4, w, positions=w),
                lambda: paged.paged_evict(cache, t, n, 4, w, keep_from=n[:1]),
                lambda: paged.paged_append(cache, k[0], k[0], t, n, n),
                lambda: paged.paged_append(cache, q[:, :2], q[:2, :2], t, n, torch.zeros(4, **i32)),
                lambda: paged.paged_append(cache, q[:, :2], q[:, :2], t, n, n)):
        with pytest.raises(ValueError):
            bad()


def test_attention_shapes_one_after_another():
    """Calls of different shapes share the scratch: none finds what another
    left in it."""
    rng = np.random.default_rng(20)
    runs = []
    for heads, d, lengths in ((1, 128, [30000]), (4, 64, [500] * 300), (2, 256, [9000, 1, 4000]), (8, 64, [3] * 400)):
        lengths = np.asarray(lengths, dtype=np.int32)
        table, pages = ref.page_table(lengths, 64, rng)
        k, v = (torch.randn(pages, heads, 64, d, device="cuda").bfloat16() for _ in range(2))
        q = torch.randn(len(lengths), 8, d, device="cuda").bfloat16()
        args = (paged.PagedKV(k, v), q, torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda())
        runs.append((args, paged.paged_attn_decode(*args)))
    for _ in range(3):
        for args, first in runs:
            assert torch.equal(paged.paged_attn_decode(*args), first) and bool(torch.isfinite(first).all())
