"""Attention whose weights span many powers of two: one slot in sixteen takes
almost all of the softmax and has a V of zero, so the output is what the other
slots, each 2^-20 to 2^-26 of it, bring.

Bounds.  Scores are exact here (one dim of q is 1, the others 0), so a weight
is off by the rounding of x * scale * log2(e), below 2^-17 of it, and by ex2's
2^-22; the MMA's sums add a few 2^-23 each: 2^-14 of sum p |v| covers them.
The weights (times the slot's scale for codes) enter the PV product as two
fp16 numbers, in units where the largest of them is at least 2^9, on a grid of
2^-24 at the finest: an error of 2^-34 of that largest one per slot, or 2^-22 of
the product itself.  Last the output is rounded: 2^-11 (fp16) or 2^-8 (bf16) of
the value."""
import numpy as np
import pytest
import torch

from rec_b200 import paged
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

PAGE = 16
LENGTHS = np.array([4097, 40, 1000, 17], dtype=np.int32)
SCALE = float(np.float32(np.log(2.0)))  # scores of K's first dim in powers of two


def slots_of(table):
    """(page, offset) of every attended slot, and whether it dominates."""
    at = [ref.rows_of(table, b, n, PAGE) for b, n in enumerate(LENGTHS)]
    first = [np.arange(n) % 16 == 5 for n in LENGTHS]
    return np.concatenate([p for p, _ in at]), np.concatenate([o for _, o in at]), np.concatenate(first)


def run(cache, K, V, table, unit, heads, spread, dtype, group=8):
    """spread[page, offset, dim]: the finest step of a slot's product with its
    V, that is the largest |v| or |code| that multiplies the weight's error."""
    d = cache.head_dim
    q = torch.zeros(len(LENGTHS), heads * group, d, device="cuda", dtype=dtype)
    q[:, :, 0] = 1.0
    lse = torch.empty(len(LENGTHS), heads * group, device="cuda")
    out = paged.paged_attn_decode(cache, q, torch.from_numpy(table).cuda(), torch.from_numpy(LENGTHS).cuda(), scale=SCALE,
                                  lse=lse).double().cpu().numpy()
    paged.check_status()
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    for b, n in enumerate(LENGTHS):
        pg, off = ref.rows_of(table, b, n, PAGE)
        for h in range(heads):
            s = K[pg, h, off, 0] * SCALE
            p = np.exp(s - s.max())
            total = p.sum()
            v = V[pg, h, off]
            want = (p @ v) / total
            top = (p * unit[pg, h, off]).max()  # the largest product
            bound = (u * np.abs(want) + (2.0 ** -14 * (p @ np.abs(v)) + 2.0 ** -34 * top * spread[pg, h, off].sum(0)) / total
                     + (2.0 ** -25 if dtype == torch.float16 else 0.0))
            got = out[b, h * group:(h + 1) * group]
            assert (np.abs(got - want) <= bound).all(), (b, h, np.abs(got - want).max(), bound.min(), want.max())
            assert np.abs(lse[b, h * group:(h + 1) * group].double().cpu().numpy() - s.max() - np.log(total)).max() <= 1e-5


@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("tail", [3.0, 20.3, 22.3, 24.5, 25.5])
@pytest.mark.parametrize("d", [64, 128])
def test_rows(kind, tail, d):
    rng = np.random.default_rng(int(10 * tail))
    dt = torch.float16 if kind == "fp16" else torch.bfloat16
    table, pages = ref.page_table(LENGTHS, PAGE, rng)
    pg, off, big = slots_of(table)
    heads = 2
    k = np.full((pages, heads, PAGE, d), 3.0, dtype=np.float32)
    v = 2.0 ** 12 * (1 + 0.25 * rng.standard_normal((pages, heads, PAGE, d))).astype(np.float32)
    k[pg, :, off, 0] = np.where(big, 0.0, -tail)[:, None]
    v[pg[big], :, off[big]] = 0.0
    k, v = (torch.from_numpy(x).cuda().to(dt) for x in (k, v))
    V = ref.values(v, 16)
    run(paged.PagedKV(k, v), ref.values(k, 16), V, table, np.ones(V.shape[:3]), heads, np.abs(V), dt)


@pytest.mark.parametrize("kb,vb", [(8, 8), (8, 4), (4, 8), (4, 4)])
@pytest.mark.parametrize("code", [4, 2, 0])
@pytest.mark.parametrize("wide", [0, 6, -20])
@pytest.mark.parametrize("d", [64, 256])
def test_codes(kb, vb, code, wide, d):
    """wide: the dominating slots' scale is 2^wide times the others' (their
    value is zero all the same: bias = -middle * scale)."""
    rng = np.random.default_rng(100 * kb + 10 * vb + code)
    table, pages = ref.page_table(LENGTHS, PAGE, rng)
    pg, off, big = slots_of(table)
    heads, groups = 2, d // 64
    shape = (pages, heads, PAGE)
    # K: -26.25 .. 0 in steps of 1.75 (4 bits), or the same from every 14th code of 8 bits
    ks, kbias, top = (1.75, -26.25, 15) if kb == 4 else (0.125, -26.25, 210)
    kc = rng.integers(0, 1 << kb, (*shape, d))
    kc[pg, :, off, 0] = np.where(big, top, code if kb == 4 else 14 * code)[:, None]
    mid = 1 << (vb - 1)
    vc = rng.integers(0, 1 << vb, (*shape, d))
    vc[pg[big], :, off[big]] = mid
    s = np.full((*shape, groups), 1.296875, dtype=np.float32)
    s *= 2.0 ** rng.integers(-3, 4, s.shape)
    bias = s * 8
    s[pg[big], :, off[big]] = 2.0 ** wide
    bias[pg[big], :, off[big]] = -mid * 2.0 ** wide

    def bf(x):
        return torch.from_numpy(np.ascontiguousarray(np.broadcast_to(x, (*shape, groups))).astype(np.float32)).cuda().bfloat16()

    k, v = ref.pack(kc, kb).cuda(), ref.pack(vc, vb).cuda()
    scales = [bf(ks), bf(kbias), bf(s), bf(bias)]
    cache = paged.PagedKV(k, v, *scales)
    unit = np.abs(scales[2].double().cpu().numpy())
    # a product's error times |code - middle|
    run(cache, ref.values(k, kb, *scales[:2]), ref.values(v, vb, *scales[2:]), table, unit.max(-1), heads,
        np.abs(vc - mid).astype(np.float64), torch.bfloat16)
