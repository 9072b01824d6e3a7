// Paged cache: argument checks and the append.
#include <limits.h>

#include "paged.cuh"
#include "quant.cuh"

using namespace rec;

namespace rec {

int paged_view(const RecPagedKV* kv, const RecPagedTable* table, const char* who, PagedView* out) {
  REC_CHECK_ARG(kv && table, "%s: null cache or table", who);
  REC_CHECK_ARG(table->table && (reinterpret_cast<uintptr_t>(table->table) & 3u) == 0,
                "%s: the page table must be non-null and 4-byte aligned", who);
  REC_CHECK_ARG(table->batch >= 1 && table->batch <= 4096, "%s: batch %d outside 1..4096", who, table->batch);
  REC_CHECK_ARG(table->width >= 1 && table->table_stride >= table->width, "%s: bad page table width %d or stride", who,
                table->width);
  REC_CHECK_ARG(kv->n_pages >= 1 && kv->page_size >= 1 && kv->page_size <= 65536 && kv->n_kv_heads >= 1 &&
                    kv->n_kv_heads <= 1024,
                "%s: bad pool shape (%d pages of %d rows, %d kv heads)", who, kv->n_pages, kv->page_size,
                kv->n_kv_heads);
  const int64_t slots = int64_t(table->width) * kv->page_size;
  REC_CHECK_ARG(slots <= INT_MAX - 65536, "%s: a page table of %lld slots", who, (long long)slots);
  const bool wide = kv->k_bits == 16 && kv->v_bits == 16;
  const bool codes = (kv->k_bits == 8 || kv->k_bits == 4) && (kv->v_bits == 8 || kv->v_bits == 4);
  REC_CHECK_ARG(wide || codes, "%s: K and V bits must both be 16, or each 8 or 4 (got %d, %d)", who, kv->k_bits,
                kv->v_bits);
  REC_CHECK_ARG(kv->dtype == REC_T_BF16 || (wide && kv->dtype == REC_T_FP16),
                "%s: rows are bf16 or fp16 (quantized caches: bf16)", who);
  REC_CHECK_ARG(codes ? kv->head_dim == 64 || kv->head_dim == 128 || kv->head_dim == 256
                      : kv->head_dim >= 8 && kv->head_dim <= 256 && kv->head_dim % 8 == 0,
                "%s: head_dim %d must be a multiple of 8 up to 256 (codes: 64, 128 or 256)", who, kv->head_dim);
  PagedView& p = *out;
  const int d = kv->head_dim;
  const int64_t n[3] = {kv->n_pages, kv->n_kv_heads, kv->page_size};
  for (int i = 0; i < 2; ++i) {
    void* base = i ? kv->v : kv->k;
    const int64_t* st = i ? kv->v_stride : kv->k_stride;
    const int bits = i ? kv->v_bits : kv->k_bits;
    REC_CHECK_ARG(base && aligned16(base), "%s: %s must be non-null and 16-byte aligned", who, i ? "V" : "K");
    int64_t span = int64_t(d) * bits / 8;
    for (int j = 0; j < 3; ++j) {
      if (n[j] == 1) continue;  // never stepped over
      REC_CHECK_ARG(st[j] >= 0 && st[j] % 16 == 0 && st[j] < (int64_t(1) << 36),
                    "%s: %s strides must be non-negative multiples of 16 bytes", who, i ? "V" : "K");
      span += st[j] * (n[j] - 1);  // n < 2^31, st < 2^36: no overflow
    }
    REC_CHECK_ARG(span <= (int64_t(1) << 36), "%s: the %s pool spans more than 64 GB", who, i ? "V" : "K");
    (i ? p.v : p.k) = {static_cast<uint8_t*>(base), uint32_t(st[0] >> 4), uint32_t(st[1] >> 4), uint32_t(st[2] >> 4)};
    if (!codes) {
      (i ? p.vs : p.ks) = {};
      continue;
    }
    void* s = i ? kv->v_scales : kv->k_scales;
    void* b = i ? kv->v_biases : kv->k_biases;
    const int64_t* ss = i ? kv->v_scale_stride : kv->k_scale_stride;
    const int rb = d / 32;  // bytes of a row's scales
    REC_CHECK_ARG(s && b && reinterpret_cast<uintptr_t>(s) % rb == 0 && reinterpret_cast<uintptr_t>(b) % rb == 0,
                  "%s: scales and biases must be non-null and %d-byte aligned", who, rb);
    span = rb;
    for (int j = 0; j < 3; ++j) {
      if (n[j] == 1) continue;
      REC_CHECK_ARG(ss[j] >= 0 && ss[j] % rb == 0 && ss[j] < (int64_t(1) << 33),
                    "%s: scale strides must be non-negative multiples of %d bytes", who, rb);
      span += ss[j] * (n[j] - 1);
    }
    REC_CHECK_ARG(span <= (int64_t(1) << 33), "%s: the scales span more than 8 GB", who);
    (i ? p.vs : p.ks) = {static_cast<uint16_t*>(s), static_cast<uint16_t*>(b), uint32_t(ss[0] >> 1),
                         uint32_t(ss[1] >> 1), uint32_t(ss[2] >> 1)};
  }
  p.n_pages = kv->n_pages;
  p.hkv = kv->n_kv_heads;
  p.d = d;
  p.k_bits = kv->k_bits;
  p.v_bits = kv->v_bits;
  p.fp16 = kv->dtype == REC_T_FP16;
  p.ps = make_fastdiv(uint32_t(kv->page_size));
  p.table = table->table;
  p.table_stride = table->table_stride;
  p.width = table->width;
  p.batch = table->batch;
  p.slots = slots;
  return REC_OK;
}

}  // namespace rec

namespace {

// ---------------------------------------------------------------------------
// Append.  16-bit rows are bound by their bytes (16 prompts, 282 MB: 49.8 us,
// 5.65 TB/s), codes by the quantisation's arithmetic (16 x 4,096 tokens of 8
// bit: 113 us, 1.8 TB/s), a decode step by latency (64 tokens of 8 bit: 3.9
// us).  A row's place (session by bisection of cu, page by the table) is found
// once, by one thread, for all the threads that move the row.

struct AppendArgs {
  const uint16_t *k, *v;
  int64_t k_stride, v_stride, rows;
  const int *cu, *starts;
  float* weights;
  int* positions;
  const int* first;  // position of every session's first row, or NULL: its slot
  int* status;
};

// The session of row r: the last b with cu[b] <= r (cu ascending).
__device__ __forceinline__ int row_session(const int* cu, int batch, int64_t r) {
  int lo = 0, hi = batch;  // cu[lo] <= r < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= r) lo = mid; else hi = mid;
  }
  return lo;
}

// Where row r goes; page -1: nowhere (reported by the caller's first block of
// threads that looks, `tell`).
struct RowPlace {
  int page, off, position;
};
__device__ __forceinline__ RowPlace place_row(const PagedView& p, const AppendArgs& a, int64_t r, bool tell) {
  RowPlace w = {-1, 0, 0};
  const int b = row_session(a.cu, p.batch, r);
  const int c0 = __ldg(a.cu + b), c1 = __ldg(a.cu + b + 1);
  if (r < c0 || r >= c1) return w;  // cu does not cover the row
  const int64_t slot = int64_t(__ldg(a.starts + b)) + (r - c0);
  const bool inside = slot >= 0 && slot < p.slots;
  if (inside) w.page = slot_page(p, b, int(slot), w.off);
  w.position = a.first ? int(__ldg(a.first + b) + (r - c0)) : int(slot);
  if (w.page < 0 && tell) report(a.status, inside ? kStatusBadPage : kStatusBadPosition);
  return w;
}
// The new slots' weight and position, one (row, head) per lane.
__device__ __forceinline__ void mark_slots(const PagedView& p, const AppendArgs& a, const RowPlace& w, int h) {
  if (w.page < 0) return;
  const int64_t at = slot_index(p, w.page, h, w.off);
  if (a.weights) a.weights[at] = 0.0f;
  if (a.positions) a.positions[at] = w.position;
}

constexpr int kAppendThreads = 256;

// The code of w (quant_code's) with one multiplication: the product is within
// 2e-4 of the quotient (at most 255, errors of a few 2^-24), so both round to
// the same integer unless the product is that near to a half; then it divides.
__device__ __forceinline__ uint32_t near_code(float w, const QGroupParams& p, float inv, float bins) {
  const float y = __fmul_rn(__fsub_rn(w, p.bias), inv);
  float n = rintf(y);
  if (!(fabsf(fabsf(__fsub_rn(y, n)) - 0.5f) > 2e-4f)) n = rintf(__fdiv_rn(__fsub_rn(w, p.bias), p.scale));
  return uint32_t(n < 0.0f ? 0.0f : (n > bins ? bins : n));
}

// A lane's 8 values of a 64-dim group that 8 neighbouring lanes hold: its
// codes to dst (piece e of the row), and the group's scale and bias.
__device__ __forceinline__ void store_codes(const uint4& val, int bits, uint8_t* row, int e, const PagedScales& sc,
                                            size_t at) {
  const int lane = threadIdx.x & 31;
  const unsigned mask = 0xFFu << (lane & 24);
  const uint32_t w[4] = {val.x, val.y, val.z, val.w};
  float v[8], mx, mn;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf(uint16_t(w[i] & 0xFFFFu));
    v[2 * i + 1] = bf(uint16_t(w[i] >> 16));
  }
  mx = mn = v[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    mx = fmaxf(mx, v[i]);
    mn = fminf(mn, v[i]);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    mx = fmaxf(mx, __shfl_xor_sync(mask, mx, o));
    mn = fminf(mn, __shfl_xor_sync(mask, mn, o));
  }
  const QGroupParams q = group_params(mx, mn, bits);
  const float inv = __fdividef(1.0f, q.scale), bins = float((1 << bits) - 1);
  uint32_t lo = 0, hi = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = near_code(v[i], q, inv, bins);
    if (bits == 4) lo |= c << (4 * i);
    else if (i < 4) lo |= c << (8 * i);
    else hi |= c << (8 * (i - 4));
  }
  if (bits == 4) reinterpret_cast<uint32_t*>(row)[e] = lo;
  else reinterpret_cast<uint2*>(row)[e] = make_uint2(lo, hi);
  if ((lane & 7) == 0) {
    sc.s[at + (e >> 3)] = to_bf(q.scale);
    sc.b[at + (e >> 3)] = to_bf(q.bias);
  }
}

// A block takes ROWS rows at a time: their places once into shared memory,
// then every thread moves 16-byte pieces of 8 values, U on their way at once
// (codes: the 8 lanes of a group meet for its extremes).  A row's pieces: K
// heads, then V heads.
template <int ROWS, bool CODES>
__global__ void __launch_bounds__(kAppendThreads) k_append_rows(const PagedView p, const AppendArgs a, const FastDiv per,
                                                                const FastDiv line) {
  __shared__ RowPlace place[ROWS];
  const int heads_pieces = per.d;  // pieces of a row's K (as many of its V)
  for (int64_t r0 = int64_t(blockIdx.x) * ROWS; r0 < a.rows; r0 += int64_t(gridDim.x) * ROWS) {
    const int rows = int(min(int64_t(ROWS), a.rows - r0));
    if (threadIdx.x < rows) place[threadIdx.x] = place_row(p, a, r0 + threadIdx.x, true);
    __syncthreads();
    const int pieces = rows * 2 * heads_pieces;
    constexpr int U = 2;  // 49.8 us for 282 MB of prompts; 54.6 with 4, 53.5 with 8
    for (int x0 = threadIdx.x; x0 < pieces; x0 += U * kAppendThreads) {
      uint4 val[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int x = x0 + i * kAppendThreads;
        if (x >= pieces) break;
        const int half = int(fdiv(x, per)), c = x - half * heads_pieces;  // half: 2 row + (V)
        const uint16_t* src = half & 1 ? a.v + (r0 + (half >> 1)) * a.v_stride : a.k + (r0 + (half >> 1)) * a.k_stride;
        val[i] = __ldcs(reinterpret_cast<const uint4*>(src) + c);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int x = x0 + i * kAppendThreads;
        if (x >= pieces) break;
        const int half = int(fdiv(x, per)), c = x - half * heads_pieces;
        const RowPlace w = place[half >> 1];
        if (w.page < 0) continue;  // codes: all 8 lanes of a group
        const int h = int(fdiv(c, line)), e = c - h * int(line.d);
        uint8_t* row = row_ptr(half & 1 ? p.v : p.k, w.page, h, w.off);
        if constexpr (CODES) {
          const PagedScales& sc = half & 1 ? p.vs : p.ks;
          store_codes(val[i], half & 1 ? p.v_bits : p.k_bits, row, e, sc, scale_at(sc, w.page, h, w.off));
        } else {
          reinterpret_cast<uint4*>(row)[e] = val[i];
        }
      }
    }
    if (a.weights || a.positions)
      for (int x = threadIdx.x; x < rows * p.hkv; x += kAppendThreads) mark_slots(p, a, place[x / p.hkv], x % p.hkv);
    __syncthreads();
  }
}

template <bool CODES>
void launch_append(const PagedView& p, const AppendArgs& a, cudaStream_t st) {
  const FastDiv per = make_fastdiv(unsigned(p.hkv * p.d / 8)), piece = make_fastdiv(unsigned(p.d / 8));
  const int64_t most = int64_t(sm_count()) * 8;
  // few rows: a block per row, so that every SM has one; many: 8 a block share the places' latency
  if (a.rows <= 2 * most) {
    k_append_rows<1, CODES><<<unsigned(a.rows), kAppendThreads, 0, st>>>(p, a, per, piece);
  } else {
    const int64_t blocks = (a.rows + 7) / 8;
    k_append_rows<8, CODES><<<unsigned(blocks < most ? blocks : most), kAppendThreads, 0, st>>>(p, a, per, piece);
  }
}

}  // namespace

REC_API int rec_paged_append(const RecPagedKV* kv, const RecPagedTable* table, const void* k_dev, const void* v_dev,
                             int64_t k_row_stride, int64_t v_row_stride, int64_t rows, const int32_t* cu_dev,
                             const int32_t* starts_dev, float* weights, int32_t* positions,
                             const int32_t* first_positions_dev, int32_t* status_dev, void* stream) {
  PagedView p;
  const int rc = paged_view(kv, table, "rec_paged_append", &p);
  if (rc) return rc;
  REC_CHECK_ARG(rows >= 0 && rows <= INT_MAX, "rec_paged_append: bad row count %lld", (long long)rows);
  REC_CHECK_ARG(cu_dev && starts_dev, "rec_paged_append: null cu or starts");
  if (rows == 0) return REC_OK;
  const int64_t line = int64_t(p.hkv) * p.d;
  REC_CHECK_ARG(k_dev && v_dev && aligned16(k_dev) && aligned16(v_dev),
                "rec_paged_append: k and v must be non-null and 16-byte aligned");
  REC_CHECK_ARG(k_row_stride >= line && v_row_stride >= line && k_row_stride % 8 == 0 && v_row_stride % 8 == 0,
                "rec_paged_append: row strides must be multiples of 8 elements and hold a row");
  AppendArgs a = {static_cast<const uint16_t*>(k_dev), static_cast<const uint16_t*>(v_dev), k_row_stride, v_row_stride,
                  rows, cu_dev, starts_dev, weights, positions, first_positions_dev, status_dev};
  if (p.k_bits == 16) launch_append<false>(p, a, static_cast<cudaStream_t>(stream));
  else launch_append<true>(p, a, static_cast<cudaStream_t>(stream));
  REC_CHECK_CUDA(cudaGetLastError());
  return REC_OK;
}
