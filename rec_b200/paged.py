"""Batched decode over a paged key-value cache: append, attention of one new
token per session, eviction by accumulated attention weight.

A pool holds pages of `page_size` rows of every kv head; session b's slot t is
row t % page_size of page table[b, t / page_size].  Pools are torch tensors
that the caller allocates; these calls keep no reference to them.  They are
ordered on torch's current stream and do not synchronise.  A page id outside
the pool or a slot outside the table is left out and recorded on the device:
`check_status` raises for it.

Scratch memory is kept per (device, stream) and grows with the largest call,
so calls on different streams do not meet; a call under stream capture takes
its scratch from the capture's own pool.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import abi
from ._lib import check, lib

_TYPES = {torch.bfloat16: abi.REC_T_BF16, torch.float16: abi.REC_T_FP16}
_status: dict[int, torch.Tensor] = {}  # one word per device
_scratch: dict[tuple, torch.Tensor] = {}  # (call, device, stream)


class PagedKV:
    """The pools of one layer.

    16 bit: k, v bf16 or fp16 [pages, kv heads, page_size, head_dim].
    Affine group-64 codes (the formats of rec_kv_append, K and V each 8 or 4
    bits): k, v int32 words [pages, kv heads, page_size, head_dim * bits / 32]
    with bf16 scales and biases [pages, kv heads, page_size, head_dim / 64].
    Only the last dimension has to be contiguous; row starts are 16-byte
    aligned.  A view: the tensors stay the caller's."""

    __slots__ = ("k", "v", "scales", "device", "dtype", "shape", "head_dim", "desc", "_ref")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor | None = None,
                 k_biases: torch.Tensor | None = None, v_scales: torch.Tensor | None = None,
                 v_biases: torch.Tensor | None = None):
        scales = (k_scales, k_biases, v_scales, v_biases)
        kd, vd = k.shape, v.shape
        if len(kd) != 4 or len(vd) != 4 or kd[:3] != vd[:3] or not k.is_cuda or k.device != v.device:
            raise ValueError("k and v must be CUDA tensors [pages, kv heads, page_size, ...] of the same pages")
        d = abi.RecPagedKV()
        ks, vs = k.stride(), v.stride()
        if ks[3] != 1 or vs[3] != 1:
            raise ValueError("the rows of k and v must be contiguous")
        if k.dtype in _TYPES:
            if v.dtype != k.dtype or kd != vd or any(t is not None for t in scales):
                raise ValueError("16-bit pools: k and v of one type and shape, no scales")
            self.head_dim, self.dtype, item = kd[3], k.dtype, 2
            d.k_bits = d.v_bits = 16
            d.dtype = _TYPES[k.dtype]
        else:
            if k.element_size() != 4 or v.element_size() != 4 or any(t is None for t in scales):
                raise ValueError("pools must be bf16, fp16, or 32-bit code words with scales and biases")
            groups = k_scales.shape[-1]
            self.head_dim, self.dtype, item = 64 * groups, torch.bfloat16, 4
            for t, like in zip(scales, (k_scales, k_scales, v_scales, v_scales)):
                if t.dtype != torch.bfloat16 or t.shape != (*kd[:3], groups) or t.device != k.device \
                        or t.stride() != like.stride() or t.stride(3) != 1:
                    raise ValueError("scales and biases must be bf16 [pages, kv heads, page_size, head_dim / 64], "
                                     "those of one tensor with the same strides")
            if groups < 1 or kd[3] % (2 * groups) or vd[3] % (2 * groups):
                raise ValueError("code words do not match the scales' head_dim")
            d.k_bits, d.v_bits = kd[3] // (2 * groups), vd[3] // (2 * groups)
            d.dtype = abi.REC_T_BF16
            a, b = k_scales.stride(), v_scales.stride()
            d.k_scale_stride[:] = (2 * a[0], 2 * a[1], 2 * a[2])
            d.v_scale_stride[:] = (2 * b[0], 2 * b[1], 2 * b[2])
            d.k_scales, d.k_biases = k_scales.data_ptr(), k_biases.data_ptr()
            d.v_scales, d.v_biases = v_scales.data_ptr(), v_biases.data_ptr()
        d.k, d.v = k.data_ptr(), v.data_ptr()
        d.k_stride[:] = (item * ks[0], item * ks[1], item * ks[2])
        d.v_stride[:] = (item * vs[0], item * vs[1], item * vs[2])
        d.n_pages, d.n_kv_heads, d.page_size = kd[0], kd[1], kd[2]
        d.head_dim = self.head_dim
        self.k, self.v, self.scales, self.device = k, v, scales, k.device
        self.shape = tuple(kd[:3])
        self.desc = d
        self._ref = C.byref(d)

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, *, k_bits: int = 16, v_bits: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedKV":
        """Pools of `pages` pages, not cleared (every slot is written before
        it is attended)."""
        lead = (pages, kv_heads, page_size)
        if k_bits == 16 and v_bits == 16:
            return cls(*(torch.empty(*lead, head_dim, dtype=dtype, device=device) for _ in range(2)))
        if k_bits not in (4, 8) or v_bits not in (4, 8) or head_dim % 64:
            raise ValueError("K and V bits must both be 16, or each 8 or 4 with head_dim a multiple of 64")
        codes = [torch.empty(*lead, head_dim * b // 32, dtype=torch.int32, device=device) for b in (k_bits, v_bits)]
        return cls(*codes, *(torch.empty(*lead, head_dim // 64, dtype=torch.bfloat16, device=device)
                             for _ in range(4)))


def _stream(device: torch.device) -> int:
    if device.index != torch.cuda.current_device():
        raise ValueError("the tensors must live on the current CUDA device")
    return torch.cuda.current_stream(device).cuda_stream


def _status_ptr(device: torch.device) -> int | None:
    t = _status.get(device.index)
    if t is None:
        if torch.cuda.is_current_stream_capturing():
            return None  # cleared by every replay if it were captured
        t = _status[device.index] = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()  # zero before any other stream's call
    return t.data_ptr()


def _workspace(call: str, device: torch.device, stream: int, need: int) -> torch.Tensor:
    """At least `need` bytes, zero when new."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(need, dtype=torch.uint8, device=device)
    key = (call, device.index, stream)
    t = _scratch.get(key)
    if t is None or t.numel() < need:
        t = _scratch[key] = torch.zeros(need, dtype=torch.uint8, device=device)
    return t


def check_status(device=None) -> None:
    """Synchronises the device and raises RecError if a call since the last
    check met a bad page id or slot; clears the record."""
    index = torch.device("cuda" if device is None else device).index
    index = torch.cuda.current_device() if index is None else index
    t = _status.get(index)
    if t is None:
        return
    torch.cuda.synchronize(index)
    code = int(t.item())
    if code:
        t.zero_()
        check(code)


def _table(table: torch.Tensor, device: torch.device) -> abi.RecPagedTable:
    if table.dtype != torch.int32 or table.dim() != 2 or table.device != device or table.stride(1) != 1:
        raise ValueError("the page table must be int32 [batch, pages] on the cache's device, rows contiguous")
    return abi.RecPagedTable(table.data_ptr(), table.stride(0), table.shape[1], table.shape[0])


def _ints(name: str, t: torch.Tensor, n: int, device: torch.device) -> int:
    if t.dtype != torch.int32 or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor [{n}] on the cache's device")
    return t.data_ptr()


def _per_slot(name: str, t: torch.Tensor, cache: PagedKV, dtype: torch.dtype) -> int:
    if t.dtype != dtype or tuple(t.shape) != cache.shape or t.device != cache.device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor [pages, kv heads, page_size] on the cache's device")
    return t.data_ptr()


def paged_append(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
                 cu_seqlens: torch.Tensor, weights: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None) -> None:
    """Writes the new tokens' rows k, v [rows, kv heads, head_dim] (K already
    RoPE'd): row r of session b, cu_seqlens[b] <= r < cu_seqlens[b + 1], goes
    to slot starts[b] + r - cu_seqlens[b].  Quantized caches take the codes of
    rec_kv_append.  weights (fp32) and positions (int32), one value per slot:
    the written slots get 0 and their slot number."""
    dev = cache.device
    t = _table(table, dev)
    B, line = t.batch, (cache.shape[1], cache.head_dim)
    for name, x in (("k", k), ("v", v)):
        if x.dtype != cache.dtype or x.dim() != 3 or tuple(x.shape[1:]) != line or x.device != dev \
                or x.stride(2) != 1 or x.stride(1) != line[1]:
            raise ValueError(f"{name} must be {cache.dtype} [rows, {line[0]}, {line[1]}] on the cache's device, "
                             "each row contiguous")
    if k.shape[0] != v.shape[0]:
        raise ValueError("k and v must have the same rows")
    if k.shape[0] == 0:
        return
    check(lib().rec_paged_append(
        cache._ref, C.byref(t), k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), k.shape[0],
        _ints("cu_seqlens", cu_seqlens, B + 1, dev), _ints("starts", starts, B, dev),
        None if weights is None else _per_slot("weights", weights, cache, torch.float32),
        None if positions is None else _per_slot("positions", positions, cache, torch.int32),
        _status_ptr(dev), _stream(dev)), "rec_paged_append")


def paged_attn_decode(cache: PagedKV, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
                      scale: float | None = None, softcap: float = 0.0, window: int = 0,
                      sinks: torch.Tensor | None = None, out: torch.Tensor | None = None,
                      lse: torch.Tensor | None = None, weights: torch.Tensor | None = None,
                      weights_out: torch.Tensor | None = None, decay: float = 1.0) -> torch.Tensor:
    """Attention of one new token per session, q [batch, query heads,
    head_dim] over the session's lengths[b] slots; returns out, like q.

    Scores are scale (default head_dim ** -0.5) * q . k, capped as softcap *
    tanh(s / softcap) when softcap > 0; window > 0 attends the last `window`
    slots only; sinks (bf16 [query heads]) join the softmax's denominator.  A
    session with no slot gives zeros.  lse (fp32 [batch, query heads], natural
    log) is filled when given.  weights (fp32, one value per slot) accumulate:
    weights_out = decay * weights + the slot's softmax weights summed over the
    kv head's query heads, for every slot below the session's length;
    weights_out defaults to weights (in place)."""
    dev = cache.device
    t = _table(table, dev)
    B, d = t.batch, cache.head_dim
    if q.dtype != cache.dtype or q.dim() != 3 or q.shape[0] != B or q.shape[2] != d or q.device != dev \
            or q.stride(2) != 1:
        raise ValueError(f"q must be {cache.dtype} [{B}, query heads, {d}] on the cache's device, rows contiguous")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif out.dtype != q.dtype or out.shape != q.shape or out.device != dev or out.stride(2) != 1:
        raise ValueError("out must match q, rows contiguous")
    hq = q.shape[1]
    a = abi.RecPagedAttn()
    a.q, a.q_batch_stride, a.q_head_stride = q.data_ptr(), q.stride(0), q.stride(1)
    a.out, a.out_batch_stride, a.out_head_stride = out.data_ptr(), out.stride(0), out.stride(1)
    a.lengths = _ints("lengths", lengths, B, dev)
    a.n_q_heads = hq
    a.scale = d ** -0.5 if scale is None else scale
    a.softcap, a.window = softcap, window
    if lse is not None:
        if lse.dtype != torch.float32 or lse.shape != (B, hq) or lse.device != dev or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous fp32 tensor [{B}, {hq}] on the cache's device")
        a.lse = lse.data_ptr()
    if sinks is not None:
        if sinks.dtype != torch.bfloat16 or sinks.shape != (hq,) or sinks.device != dev or not sinks.is_contiguous():
            raise ValueError(f"sinks must be a contiguous bf16 tensor [{hq}] on the cache's device")
        a.sinks = sinks.data_ptr()
    if weights is not None:
        a.weights_in = _per_slot("weights", weights, cache, torch.float32)
        a.weights_out = a.weights_in
    if weights_out is not None:
        a.weights_out = _per_slot("weights_out", weights_out, cache, torch.float32)
    a.decay = decay if weights is not None else 0.0
    tr = C.byref(t)
    zero = C.c_size_t()
    need = lib().rec_paged_attn_workspace_bytes(cache._ref, tr, hq, a.weights_out is not None, C.byref(zero))
    stream = _stream(dev)
    ws = _workspace("attn", dev, stream, max(need, 256))
    counters = _workspace("attn counters", dev, stream, max(zero.value, 4096))  # every call leaves them zero
    check(lib().rec_paged_attn_decode(cache._ref, tr, C.byref(a), ws.data_ptr(), ws.numel(), counters.data_ptr(),
                                      counters.numel(), _status_ptr(dev), stream), "rec_paged_attn_decode")
    return out


def paged_evict(cache: PagedKV, table: torch.Tensor, lengths: torch.Tensor, budget: int, weights: torch.Tensor, *,
                positions: torch.Tensor | None = None, keep_from: torch.Tensor | None = None, keep_below: int = 0,
                weights_out: torch.Tensor | None = None, positions_out: torch.Tensor | None = None,
                lengths_out: torch.Tensor | None = None) -> torch.Tensor:
    """Cuts every session's cache to at most `budget` slots and returns the
    new lengths min(lengths, budget) (int32 [batch]).

    Per session and kv head the slots rank: protected ones first (position >=
    keep_from[b], or position < keep_below), then the heaviest `weights`
    (fp32, one value per slot; NaN last), then the lowest slot.  The evicted
    slots below the budget take the kept rows at or above it, each in
    ascending order, with their weight and position; nothing else moves, so a
    cut of a few tokens moves a few rows.  The order of a session's slots is
    therefore not its tokens' order afterwards: `positions` (int32, one value
    per slot, as paged_append fills it) keeps it.  Without positions a slot
    counts as its own position.  weights_out and positions_out default to the
    inputs (in place).  The pages below the budget must not be shared with
    another session."""
    dev = cache.device
    t = _table(table, dev)
    B = t.batch
    if lengths_out is None:
        lengths_out = torch.empty(B, dtype=torch.int32, device=dev)
    a = abi.RecPagedEvict()
    a.lengths, a.lengths_out = _ints("lengths", lengths, B, dev), _ints("lengths_out", lengths_out, B, dev)
    a.budget = budget
    a.weights_in = _per_slot("weights", weights, cache, torch.float32)
    a.weights_out = a.weights_in if weights_out is None else _per_slot("weights_out", weights_out, cache, torch.float32)
    if positions is not None:
        a.positions_in = _per_slot("positions", positions, cache, torch.int32)
        a.positions_out = a.positions_in
    if positions_out is not None:
        a.positions_out = _per_slot("positions_out", positions_out, cache, torch.int32)
    if keep_from is not None:
        a.keep_from = _ints("keep_from", keep_from, B, dev)
    a.keep_below = keep_below
    tr = C.byref(t)
    need = lib().rec_paged_evict_workspace_bytes(cache._ref, tr, budget)
    stream = _stream(dev)
    ws = _workspace("evict", dev, stream, max(need, 256))
    check(lib().rec_paged_evict(cache._ref, tr, C.byref(a), ws.data_ptr(), ws.numel(), _status_ptr(dev), stream),
          "rec_paged_evict")
    return lengths_out
