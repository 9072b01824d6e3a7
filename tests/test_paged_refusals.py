"""Argument checks of the batched-decode entry points: refused before
anything is launched, so no GPU is needed (the pointers are never read)."""
import ctypes as C

import pytest
import torch

from rec_b200 import _lib, abi, paged, sampling

P = 1 << 20  # an aligned address


def kv(**over):
    d = abi.RecPagedKV(k=P, v=P, n_pages=10, page_size=16, n_kv_heads=2, head_dim=128, k_bits=16, v_bits=16)
    for s in (d.k_stride, d.v_stride):
        s[:] = (16 * 2 * 256, 16 * 256, 256)
    if over.get("k_bits", 16) != 16:
        d.k_scales = d.k_biases = d.v_scales = d.v_biases = P
        for s in (d.k_scale_stride, d.v_scale_stride):
            s[:] = (16 * 2 * 4, 16 * 4, 4)
    for name, x in over.items():
        if isinstance(x, tuple):
            getattr(d, name)[:] = x
        else:
            setattr(d, name, x)
    return d


def table(**over):
    t = abi.RecPagedTable(table=P, table_stride=8, width=8, batch=3)
    for name, x in over.items():
        setattr(t, name, x)
    return t


def attn(**over):
    a = abi.RecPagedAttn(q=P, q_batch_stride=1024, q_head_stride=128, out=P, out_batch_stride=1024, out_head_stride=128,
                         lengths=P, n_q_heads=8, scale=0.1)
    for name, x in over.items():
        setattr(a, name, x)
    return a


def run_attn(k=None, t=None, a=None, ws=P, nbytes=1 << 30, counters=P, counter_bytes=1 << 20):
    return _lib.lib().rec_paged_attn_decode(C.byref(k or kv()), C.byref(t or table()), C.byref(a or attn()), ws, nbytes,
                                            counters, counter_bytes, None, None)


def run_evict(k=None, t=None, ws=P, nbytes=1 << 30, **over):
    e = abi.RecPagedEvict(lengths=P, lengths_out=P, budget=32, weights_in=P, weights_out=P)
    for name, x in over.items():
        setattr(e, name, x)
    return _lib.lib().rec_paged_evict(C.byref(k or kv()), C.byref(t or table()), C.byref(e), ws, nbytes, None, None)


def run_append(k=None, t=None, kp=P, vp=P, ks=256, vs=256, rows=5, cu=P, starts=P):
    return _lib.lib().rec_paged_append(C.byref(k or kv()), C.byref(t or table()), kp, vp, ks, vs, rows, cu, starts, None,
                                       None, None, None, None)


BAD_CACHES = [dict(k=0), dict(v=P + 8), dict(k_bits=8), dict(k_bits=3, v_bits=3), dict(k_bits=16, v_bits=8),
              dict(head_dim=12), dict(head_dim=264), dict(head_dim=0), dict(n_pages=0), dict(page_size=0),
              dict(page_size=65537), dict(n_kv_heads=0), dict(dtype=2), dict(k_bits=8, v_bits=8, dtype=1),
              dict(k_bits=8, v_bits=8, head_dim=72), dict(k_bits=8, v_bits=8, k_scales=0),
              dict(k_bits=4, v_bits=4, v_biases=P + 2), dict(k_stride=(8192, 4096, 264)),
              dict(v_stride=(-8192, 4096, 256)), dict(k_stride=(1 << 35, 4096, 256)),
              dict(k_bits=8, v_bits=8, k_scale_stride=(128, 64, 2)),
              dict(k_bits=8, v_bits=8, v_scale_stride=(1 << 32, 64, 4))]
BAD_TABLES = [dict(table=0), dict(table=P + 2), dict(batch=0), dict(batch=4097), dict(width=0), dict(table_stride=7),
              dict(width=1 << 28, table_stride=1 << 28)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_caches(bad):
    for run in (run_attn, run_append, run_evict):
        assert run(k=kv(**bad)) == abi.REC_EINVAL
        with pytest.raises(ValueError):
            _lib.check(abi.REC_EINVAL)


@pytest.mark.parametrize("bad", BAD_TABLES, ids=str)
def test_tables(bad):
    for run in (run_attn, run_append, run_evict):
        assert run(t=table(**bad)) == abi.REC_EINVAL


@pytest.mark.parametrize("bad", [dict(q=0), dict(q=P + 8), dict(out=P + 2), dict(lengths=0), dict(n_q_heads=7),
                                 dict(n_q_heads=0), dict(scale=0.0), dict(scale=float("nan")), dict(softcap=-1.0),
                                 dict(window=-1), dict(q_head_stride=124), dict(out_batch_stride=1001),
                                 dict(weights_out=P, decay=0.5)], ids=str)
def test_attention(bad):
    assert run_attn(a=attn(**bad)) == abi.REC_EINVAL


def test_workspaces():
    zero = C.c_size_t()
    need = _lib.lib().rec_paged_attn_workspace_bytes(C.byref(kv()), C.byref(table()), 8, 1, C.byref(zero))
    assert need > 0 and zero.value == 4 * 3 * 2
    assert run_attn(counters=None) == run_attn(counter_bytes=20) == run_attn(counters=P + 2) == abi.REC_EINVAL
    assert run_attn(nbytes=need - 1, a=attn(weights_out=P)) == abi.REC_EINVAL
    assert run_attn(ws=P + 128) == abi.REC_EINVAL and run_attn(ws=None) == abi.REC_EINVAL
    assert "workspace" in _lib.last_error()
    need = _lib.lib().rec_paged_evict_workspace_bytes(C.byref(kv()), C.byref(table()), 32)
    assert run_evict(nbytes=need - 1) == abi.REC_EINVAL and run_evict(ws=P + 4) == abi.REC_EINVAL
    assert _lib.lib().rec_paged_evict_workspace_bytes(C.byref(kv()), C.byref(table()), -1) == 0


@pytest.mark.parametrize("bad", [dict(lengths=0), dict(lengths_out=0), dict(weights_in=0), dict(weights_out=0),
                                 dict(positions_in=P), dict(budget=-1), dict(keep_below=-1)], ids=str)
def test_evict(bad):
    assert run_evict(**bad) == abi.REC_EINVAL


@pytest.mark.parametrize("bad", [dict(kp=0), dict(vp=P + 8), dict(ks=255), dict(vs=260), dict(rows=-1), dict(cu=0),
                                 dict(starts=0)], ids=str)
def test_append(bad):
    assert run_append(**bad) == abi.REC_EINVAL
    assert run_append(rows=0) == abi.REC_OK


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(batch=0), dict(vocab=0), dict(stride=99), dict(out_stride=99),
                                 dict(logits=0), dict(out=0), dict(history_cap=5), dict(history_cap=1 << 18, history=P),
                                 dict(n_bias=3), dict(n_bias=8191, bias_ids=P, bias_values=P),
                                 dict(allow=P, allow_stride=3)], ids=str)
def test_logit_rules(bad):
    a = dict(logits=P, stride=100, out=P, out_stride=100, dtype=0, batch=2, vocab=100)
    r = abi.RecLogitRules()
    for name, x in bad.items():
        if name in a:
            a[name] = x
        else:
            setattr(r, name, x)
    assert _lib.lib().rec_process_logits(a["logits"], a["stride"], a["out"], a["out_stride"], a["dtype"], a["batch"],
                                         a["vocab"], C.byref(r), None) == abi.REC_EINVAL


def test_python_refuses_cpu_tensors():
    x = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        paged.PagedKV(x, x)
    with pytest.raises(ValueError):
        sampling.process_logits(torch.zeros(1, 10))


def test_packs_match_the_structures():
    def flat(t):
        return [x for n, _ in t._fields_ for x in (getattr(t, n) if hasattr(getattr(t, n), "__len__") else [getattr(t, n)])]
    for pack, kind, n in ((paged._KV, abi.RecPagedKV, 25), (paged._TABLE, abi.RecPagedTable, 4),
                          (paged._ATTN, abi.RecPagedAttn, 16), (paged._EVICT, abi.RecPagedEvict, 9),
                          (sampling._RULES, abi.RecLogitRules, 12)):
        assert flat(kind.from_buffer_copy(pack.pack(*range(1, n + 1)))) == list(range(1, n + 1))
