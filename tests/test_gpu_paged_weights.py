"""Accumulated weights at the edges: sessions whose every score is -inf, and
what the weights' kernel alone looks at."""
import numpy as np
import pytest
import torch

from rec_b200 import paged
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("group", [4, 5])
def test_scores_that_are_all_minus_infinity(dtype, group):
    """Keys that a mask holds at -inf (or at a lowest value whose products
    overflow): nothing is attended, so the output is zero, lse -inf, and the
    weights only decay."""
    heads, page, d = 2, 16, 64
    lengths = np.array([40, 40, 40], dtype=np.int32)
    table, pages = ref.page_table(lengths, page, np.random.default_rng(0))
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(pages, heads, page, d, device="cuda", generator=g).to(dtype) for _ in range(2))
    low = torch.finfo(torch.bfloat16).min if dtype == torch.bfloat16 else float("-inf")
    q = torch.ones(3, heads * group, d, device="cuda", dtype=dtype)
    for b, dead in ((0, 40), (1, 39)):  # all of them, all but the last; session 2 has none
        pg, off = ref.rows_of(table, b, dead, page)
        k[pg, :, off] = low
    w = torch.rand(pages, heads, page, device="cuda", generator=g)
    before = w.double().cpu().numpy()
    lse = torch.zeros(3, heads * group, device="cuda")
    out = paged.paged_attn_decode(paged.PagedKV(k, v), q, torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda(),
                                  lse=lse, weights=w, decay=0.5)
    paged.check_status()
    assert not out[0].any() and bool((lse[0] == float("-inf")).all())
    got = w.double().cpu().numpy()
    for b, added in ((0, np.zeros(40)), (1, np.r_[np.zeros(39), group])):
        pg, off = ref.rows_of(table, b, 40, page)
        for h in range(heads):
            assert np.abs(got[pg, h, off] - (0.5 * before[pg, h, off] + added)).max() <= 1e-5
    assert torch.equal(out[1].reshape(heads, group, d), v[table[1, 2], :, 7][:, None].expand(-1, group, -1))
    pg, off = ref.rows_of(table, 2, 40, page)
    for h in range(heads):
        assert abs((got[pg, h, off] - 0.5 * before[pg, h, off]).sum() - group) <= 1e-4


@pytest.mark.parametrize("window", [0, 20])
def test_bad_pages_below_the_window_are_reported(window):
    """The attention does not look there, the weights do: the slots are left
    out, and the call is recorded."""
    page, lengths = 16, np.array([100], dtype=np.int32)
    table, pages = ref.page_table(lengths, page, np.random.default_rng(2))
    k = torch.randn(pages, 1, page, 64, device="cuda").bfloat16()
    q = torch.randn(1, 4, 64, device="cuda").bfloat16()
    n = torch.from_numpy(lengths).cuda()
    for bad in (-1, pages):
        broken = table.copy()
        broken[0, 2] = bad
        w = torch.ones(pages, 1, page, device="cuda")
        paged.paged_attn_decode(paged.PagedKV(k, k), q, torch.from_numpy(broken).cuda(), n, window=window, weights=w,
                                decay=0.25)
        with pytest.raises(RuntimeError, match="status 5"):
            paged.check_status()
        paged.check_status()
        assert bool((w[int(table[0, 2])] == 1.0).all()) and bool((w[int(table[0, 0])] != 1.0).all())
        # without weights, what lies below the window is nobody's
        paged.paged_attn_decode(paged.PagedKV(k, k), q, torch.from_numpy(broken).cuda(), n, window=20)
        paged.check_status()
