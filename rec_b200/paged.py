"""Batched decode over a paged key-value cache: append, attention of one new
token per session, eviction by accumulated attention weight.

A pool holds pages of `page_size` rows of every kv head; session b's slot t is
row t % page_size of page table[b, t / page_size].  Pools are torch tensors
that the caller allocates; these calls keep no reference to them.  They are
ordered on torch's current stream and do not synchronise.  A page id outside
the pool or a slot outside the table is left out and recorded on the device:
`check_status` raises for it.  The record is made with a device's first
PagedKV; a graph that is captured before any was made records nothing, and the
capture warns.

Scratch memory is kept per (device, stream) for the life of the process and
grows with the largest call, so calls on different streams do not meet; a call under stream capture takes
its scratch from the capture's own pool.  Threads may share a stream: a lock
keeps one call's launches together.
"""
from __future__ import annotations

import ctypes as C
import struct
import threading
import warnings

import torch

from . import abi
from ._lib import check, lib
from .ops import current_device as _current_device, raw_stream as _raw_stream

_TYPES = {torch.bfloat16: abi.REC_T_BF16, torch.float16: abi.REC_T_FP16}
_status: dict[int, tuple] = {}  # device -> (one word, its address)
_scratch: dict[tuple, tuple] = {}  # (call, device, stream) -> (tensors, addresses and sizes)
# Held from the lookup of a call's scratch to its last launch: the library is
# called without the interpreter's lock, and another thread's call on the same
# stream would replace the scratch before this one's launch, or launch between
# this one's two kernels.
_lock = threading.Lock()
_sizes: dict[tuple, tuple] = {}  # shape of a call -> scratch bytes

# The C structures of abi.py as one pack each: a step makes these calls once
# per layer, and filling a ctypes structure field by field costs several
# microseconds of it.
_KV = struct.Struct("@6P12q7i4x")
_TABLE = struct.Struct("@Pq2i")
_ATTN = struct.Struct("@Pqq Pqq 3P i2fi 2P f4x".replace(" ", ""))
_EVICT = struct.Struct("@2Pi4x5Pi4x")
for _pack, _type in ((_KV, abi.RecPagedKV), (_TABLE, abi.RecPagedTable), (_ATTN, abi.RecPagedAttn),
                     (_EVICT, abi.RecPagedEvict)):
    assert _pack.size == C.sizeof(_type), _type

_bf16, _f32, _i32 = torch.bfloat16, torch.float32, torch.int32
_WORDS = (torch.int32, torch.uint32)  # of codes
_capturing = torch.cuda.is_current_stream_capturing


class PagedKV:
    """The pools of one layer.

    16 bit: k, v bf16 or fp16 [pages, kv heads, page_size, head_dim].
    Affine group-64 codes (the formats of rec_kv_append, K and V each 8 or 4
    bits): k, v int32 words [pages, kv heads, page_size, head_dim * bits / 32]
    with bf16 scales and biases [pages, kv heads, page_size, head_dim / 64].
    Only the last dimension has to be contiguous; row starts are 16-byte
    aligned.  A view: the tensors stay the caller's."""

    __slots__ = ("k", "v", "scales", "dtype", "shape", "head_dim", "bits", "_desc", "_index")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor | None = None,
                 k_biases: torch.Tensor | None = None, v_scales: torch.Tensor | None = None,
                 v_biases: torch.Tensor | None = None):
        dtype, index = k.dtype, k.get_device()
        if k.dim() != 4 or v.dim() != 4 or index < 0 or v.get_device() != index:
            raise ValueError("k and v must be CUDA tensors [pages, kv heads, page_size, ...]")
        pages, heads, page, kw = k.shape
        pages_v, heads_v, page_v, vw = v.shape
        if pages != pages_v or heads != heads_v or page != page_v:
            raise ValueError("k and v must have the same pages")
        k0, k1, k2, k3 = k.stride()
        v0, v1, v2, v3 = v.stride()
        if k3 != 1 or v3 != 1:
            raise ValueError("the rows of k and v must be contiguous")
        kind = _TYPES.get(dtype)
        if kind is not None:
            if v.dtype is not dtype or kw != vw \
                    or not (k_scales is None and k_biases is None and v_scales is None and v_biases is None):
                raise ValueError("16-bit pools: k and v of one type and shape, no scales")
            self.head_dim, self.dtype, self.bits = kw, dtype, (16, 16)
            self._desc = _KV.pack(k.data_ptr(), v.data_ptr(), 0, 0, 0, 0, 2 * k0, 2 * k1, 2 * k2, 2 * v0, 2 * v1, 2 * v2,
                                  0, 0, 0, 0, 0, 0, pages, page, heads, kw, 16, 16, kind)
        else:
            if dtype not in _WORDS or v.dtype not in _WORDS or k_scales is None or k_biases is None \
                    or v_scales is None or v_biases is None:
                raise ValueError("pools must be bf16, fp16, or 32-bit code words with scales and biases")
            shape, a, b = k_scales.shape, k_scales.stride(), v_scales.stride()
            if shape[:-1] != (pages, heads, page) or a[-1] != 1 or b[-1] != 1 \
                    or k_biases.shape != shape or v_scales.shape != shape or v_biases.shape != shape \
                    or k_biases.stride() != a or v_biases.stride() != b \
                    or not (k_scales.dtype is k_biases.dtype is v_scales.dtype is v_biases.dtype is _bf16) \
                    or not (k_scales.get_device() == k_biases.get_device() == v_scales.get_device()
                            == v_biases.get_device() == index):
                raise ValueError("scales and biases must be bf16 [pages, kv heads, page_size, head_dim / 64], "
                                 "those of one tensor with the same strides")
            groups = shape[3]
            if groups < 1 or kw % (2 * groups) or vw % (2 * groups):
                raise ValueError("code words do not match the scales' head_dim")
            self.head_dim, self.dtype = 64 * groups, _bf16
            self.bits = kb, vb = kw // (2 * groups), vw // (2 * groups)
            self._desc = _KV.pack(
                k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), k_biases.data_ptr(), v_scales.data_ptr(),
                v_biases.data_ptr(), 4 * k0, 4 * k1, 4 * k2, 4 * v0, 4 * v1, 4 * v2, 2 * a[0], 2 * a[1], 2 * a[2],
                2 * b[0], 2 * b[1], 2 * b[2], pages, page, heads, 64 * groups, kb, vb, abi.REC_T_BF16)
        self.k, self.v, self._index = k, v, index
        self.scales = (k_scales, k_biases, v_scales, v_biases)
        self.shape = (pages, heads, page)
        if index not in _status and not _capturing():
            _status_ptr(index)  # so that a first call under capture finds it

    @property
    def device(self) -> torch.device:
        return self.k.device

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


def _packed(pack: struct.Struct, *fields) -> bytes:
    try:
        return pack.pack(*fields)
    except struct.error as e:  # a number that the C structure's field does not hold
        raise ValueError(f"an argument is out of range: {e}") from None


def _stream(index: int) -> int:
    if index != _current_device():
        raise ValueError("the tensors must live on the current CUDA device")
    return _raw_stream(index)


def _status_ptr(index: int) -> int | None:
    s = _status.get(index)
    if s is None:
        if _capturing():  # made here it would be cleared by every replay
            warnings.warn("bad pages and slots of this capture are not recorded: make a PagedKV before it begins",
                          RuntimeWarning, stacklevel=3)
            return None
        t = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
        torch.cuda.current_stream(index).synchronize()  # zero before any other stream's call
        s = _status.setdefault(index, (t, t.data_ptr()))  # the first thread's word
    return s[1]


def _buffers(call: str, index: int, stream: int, need: int, zero: int) -> tuple:
    """The call's workspace and its counters, which are zero between calls:
    the tensors, which the caller holds until the launch, and (address, bytes,
    address, bytes).  Called with the lock held."""
    s = _scratch.get((call, index, stream))
    capturing = _capturing()
    if s is not None and s[1][1] >= need and s[1][3] >= zero and not capturing:
        return s
    device = torch.device("cuda", index)
    need, zero = max(need, 256), max(zero, 4096) if zero else 0
    if s is not None and not capturing:
        need, zero = max(need, s[1][1]), max(zero, s[1][3])
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    counters = torch.zeros(zero, dtype=torch.uint8, device=device) if zero else None
    s = ((ws, counters), (ws.data_ptr(), need, counters.data_ptr() if zero else 0, zero))
    if not capturing:
        _scratch[(call, index, stream)] = s
    return s


def check_status(device=None) -> None:
    """Synchronises the device and raises RecError if a call since the last
    check met a bad page id or slot; clears the record."""
    index = torch.device("cuda" if device is None else device).index
    index = torch.cuda.current_device() if index is None else index
    s = _status.get(index)
    if s is None:
        return
    torch.cuda.synchronize(index)
    code = int(s[0].item())
    if code:
        s[0].zero_()
        check(code)


def _table(table: torch.Tensor, index: int) -> tuple:
    """(the packed table, batch, width)."""
    if table.dtype != _i32 or table.get_device() != index or table.dim() != 2:
        raise ValueError("the page table must be int32 [batch, pages] on the cache's device, rows contiguous")
    batch, width = table.shape
    row, entry = table.stride()
    if entry != 1 and width > 1:
        raise ValueError("the page table's rows must be contiguous")
    return _TABLE.pack(table.data_ptr(), row if batch > 1 else width, width, batch), batch, width


def _ints(name: str, t: torch.Tensor, n: int, index: int) -> int:
    if t.dtype is not _i32 or t.get_device() != index or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor [{n}] on the cache's device")
    return t.data_ptr()


def _per_slot(name: str, t: torch.Tensor, cache: PagedKV, dtype: torch.dtype) -> int:
    if t.dtype != dtype or t.get_device() != cache._index or t.shape != cache.shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor [pages, kv heads, page_size] on the cache's device")
    return t.data_ptr()


def paged_append(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
                 cu_seqlens: torch.Tensor, weights: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None, first_positions: torch.Tensor | None = None) -> None:
    """Writes the new tokens' rows k, v [rows, kv heads, head_dim] (K already
    RoPE'd): row r of session b, cu_seqlens[b] <= r < cu_seqlens[b + 1], goes
    to slot starts[b] + r - cu_seqlens[b].  Quantized caches take the codes of
    rec_kv_append.  weights (fp32) and positions (int32), one value per slot:
    the written slots get 0 and their token's position, first_positions[b]
    (int32) + r - cu_seqlens[b]; without first_positions their slot number,
    which it is until the session's first eviction."""
    index = cache._index
    t, B, _ = _table(table, index)
    heads, d, dtype = cache.shape[1], cache.head_dim, cache.dtype
    rows, want = k.shape[0], (k.shape[0], heads, d)
    (k0, k1, k2), (v0, v1, v2) = k.stride(), v.stride()
    if k.dtype != dtype or v.dtype != dtype or k.shape != want or v.shape != want \
            or k.get_device() != index or v.get_device() != index or k2 != 1 or v2 != 1 or (heads > 1 and (k1 != d or v1 != d)):
        raise ValueError(f"k and v must be {dtype} [rows, {heads}, {d}] on the cache's device, each row contiguous")
    if rows == 0 or B == 0:
        return
    if rows == 1:  # a single row's stride is never used
        k0 = v0 = heads * d
    code = lib().rec_paged_append(
        cache._desc, t, k.data_ptr(), v.data_ptr(), k0, v0, rows,
        _ints("cu_seqlens", cu_seqlens, B + 1, index), _ints("starts", starts, B, index),
        None if weights is None else _per_slot("weights", weights, cache, _f32),
        None if positions is None else _per_slot("positions", positions, cache, _i32),
        None if first_positions is None else _ints("first_positions", first_positions, B, index),
        _status_ptr(index), _stream(index))
    if code:
        check(code)


def paged_attn_decode(cache: PagedKV, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
                      scale: float | None = None, softcap: float = 0.0, window: int = 0,
                      sinks: torch.Tensor | None = None, out: torch.Tensor | None = None,
                      lse: torch.Tensor | None = None, weights: torch.Tensor | None = None,
                      weights_out: torch.Tensor | None = None, decay: float = 1.0) -> torch.Tensor:
    """Attention of one new token per session, q [batch, query heads,
    head_dim] over the session's lengths[b] slots; returns out, like q.

    Scores are scale (default head_dim ** -0.5) * q . k, capped as softcap *
    tanh(s / softcap) when softcap > 0; window > 0 attends the last `window`
    slots only, which are the last tokens until the session's first eviction;
    sinks (bf16 [query heads]) join the softmax's denominator.  A session with
    no slot gives zeros.  lse (fp32 [batch, query heads], natural log, the sink
    included) is filled when given.  weights (fp32, one value per slot) accumulate:
    weights_out = decay * weights + the slot's softmax weights summed over the
    kv head's query heads, for every slot below the session's length;
    weights_out defaults to weights (in place).  Slots that take weights belong
    to one session each.  Such a call keeps a score per query head and slot of
    the page table, 4 * batch * query heads * width * page_size bytes of scratch
    whatever the lengths are: 1.07 GB for 64 sessions of 32 heads and a table of
    131,072 slots.  Slice the table to the longest session where that counts."""
    index, d = cache._index, cache.head_dim
    t, B, width = _table(table, index)
    shape = q.shape
    if q.dtype != cache.dtype or len(shape) != 3 or shape[0] != B or shape[2] != d or q.get_device() != index \
            or q.stride(2) != 1:
        raise ValueError(f"q must be {cache.dtype} [{B}, query heads, {d}] on the cache's device, rows contiguous")
    if out is None:
        out = torch.empty_like(q)
    elif out.dtype != q.dtype or out.shape != shape or out.get_device() != index or out.stride(2) != 1:
        raise ValueError("out must match q, rows contiguous")
    hq = shape[1]
    lse_at = sinks_at = weights_at = weights_to = 0
    if lse is not None:
        if lse.dtype != _f32 or lse.shape != (B, hq) or lse.get_device() != index or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous fp32 tensor [{B}, {hq}] on the cache's device")
        lse_at = lse.data_ptr()
    if sinks is not None:
        if sinks.dtype != _bf16 or sinks.shape != (hq,) or sinks.get_device() != index or not sinks.is_contiguous():
            raise ValueError(f"sinks must be a contiguous bf16 tensor [{hq}] on the cache's device")
        sinks_at = sinks.data_ptr()
    if weights is not None:
        weights_at = weights_to = _per_slot("weights", weights, cache, _f32)
    else:
        decay = 0.0
    if weights_out is not None:
        weights_to = _per_slot("weights_out", weights_out, cache, _f32)
    (q0, q1, _), (o0, o1, _) = q.stride(), out.stride()
    if B == 1:  # a single session's or head's stride is never used
        q0 = o0 = 0
    if hq == 1:
        q1 = o1 = 0
    a = _packed(_ATTN, q.data_ptr(), q0, q1, out.data_ptr(), o0, o1, lse_at, _ints("lengths", lengths, B, index), sinks_at,
                hq, d ** -0.5 if scale is None else scale, softcap, window, weights_at, weights_to, decay)
    if B == 0:
        return out
    L = lib()
    key = (index, B, width, hq, d, cache.shape, cache.bits, weights_to != 0)
    size = _sizes.get(key)
    if size is None:
        zero = C.c_size_t()
        need = L.rec_paged_attn_workspace_bytes(cache._desc, t, hq, weights_to != 0, C.byref(zero))
        size = (need, zero.value)
        if need:
            if len(_sizes) >= 4096:  # a server's batches and widths vary without end
                _sizes.clear()
            _sizes[key] = size
    stream = _stream(index)
    with _lock:
        held, at = _buffers("attn", index, stream, *size)
        code = L.rec_paged_attn_decode(cache._desc, t, a, *at, _status_ptr(index), stream)
    if code:
        check(code)
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
    index = cache._index
    t, B, _ = _table(table, index)
    if lengths_out is None:
        lengths_out = torch.empty_like(lengths)
    weights_at = weights_to = _per_slot("weights", weights, cache, _f32)
    positions_at = positions_to = keep_at = 0
    if weights_out is not None:
        weights_to = _per_slot("weights_out", weights_out, cache, _f32)
    if positions is not None:
        positions_at = positions_to = _per_slot("positions", positions, cache, _i32)
    if positions_out is not None:
        positions_to = _per_slot("positions_out", positions_out, cache, _i32)
    if keep_from is not None:
        keep_at = _ints("keep_from", keep_from, B, index)
    a = _packed(_EVICT, _ints("lengths", lengths, B, index), _ints("lengths_out", lengths_out, B, index), budget,
                weights_at, weights_to, positions_at, positions_to, keep_at, keep_below)
    if B == 0:
        return lengths_out
    L = lib()
    stream = _stream(index)
    need = L.rec_paged_evict_workspace_bytes(cache._desc, t, budget)
    with _lock:
        held, at = _buffers("evict", index, stream, need, 0)
        code = L.rec_paged_evict(cache._desc, t, a, at[0], at[1], _status_ptr(index), stream)
    if code:
        check(code)
    return lengths_out
