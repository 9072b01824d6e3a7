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
// Append.  One warp per (row, kv head, K or V).

struct AppendArgs {
  const uint16_t *k, *v;
  int64_t k_stride, v_stride, rows;
  const int *cu, *starts;
  float* weights;
  int* positions;
  int* status;
};

// The session of row r: the last b with cu[b] <= r (cu ascending).
__device__ __forceinline__ int row_session(const int* cu, int batch, int64_t r) {
  int lo = 0, hi = batch;  // cu[lo] <= r < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= r) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void k_paged_append(const PagedView p, const AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t tasks = a.rows * p.hkv * 2;
  const int64_t warps = int64_t(gridDim.x) * (blockDim.x >> 5);
  for (int64_t task = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); task < tasks; task += warps) {
    const int64_t r = task / (2 * p.hkv);
    const int rest = int(task - r * 2 * p.hkv), h = rest >> 1, is_v = rest & 1;
    const int b = row_session(a.cu, p.batch, r);
    if (r < a.cu[b] || r >= a.cu[b + 1]) continue;  // cu does not cover the row
    const int64_t slot = int64_t(a.starts[b]) + (r - a.cu[b]);
    int off = 0;
    const int page = slot >= 0 && slot < p.slots ? slot_page(p, b, int(slot), off) : -2;
    if (page < 0) {
      if (lane == 0) report(a.status, page == -1 ? kStatusBadPage : kStatusBadPosition);
      continue;
    }
    const uint16_t* src = (is_v ? a.v + r * a.v_stride : a.k + r * a.k_stride) + h * p.d;
    uint8_t* dst = row_ptr(is_v ? p.v : p.k, page, h, off);
    const int bits = is_v ? p.v_bits : p.k_bits;
    if (bits == 16) {
      for (int i = lane; i < p.d / 8; i += 32)
        reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(src)[i];
    } else {
      const PagedScales& sc = is_v ? p.vs : p.ks;
      const size_t at = scale_at(sc, page, h, off);
      const int gw = 2 * bits;  // words of a group's codes
      for (int g = 0; g < p.d / 64; ++g) {
        const uint32_t pair = reinterpret_cast<const uint32_t*>(src + 64 * g)[lane];
        const float v0 = bf(uint16_t(pair & 0xFFFFu)), v1 = bf(uint16_t(pair >> 16));
        const QGroupParams qp = warp_group_params(v0, v1, bits);
        const uint32_t word = warp_pack(quant_code(v0, qp, bits), quant_code(v1, qp, bits), bits);
        if (lane < gw) reinterpret_cast<uint32_t*>(dst)[g * gw + lane] = word;
        if (lane == 0) {
          sc.s[at + g] = to_bf(qp.scale);
          sc.b[at + g] = to_bf(qp.bias);
        }
      }
    }
    if (lane == 0 && !is_v) {
      const int64_t at = slot_index(p, page, h, off);
      if (a.weights) a.weights[at] = 0.0f;
      if (a.positions) a.positions[at] = int(slot);
    }
  }
}

}  // namespace

REC_API int rec_paged_append(const RecPagedKV* kv, const RecPagedTable* table, const void* k_dev, const void* v_dev,
                             int64_t k_row_stride, int64_t v_row_stride, int64_t rows, const int32_t* cu_dev,
                             const int32_t* starts_dev, float* weights, int32_t* positions, int32_t* status_dev,
                             void* stream) {
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
                  rows, cu_dev, starts_dev, weights, positions, status_dev};
  const int64_t warps = rows * p.hkv * 2;
  const int64_t blocks = (warps + 7) / 8, most = int64_t(sm_count()) * 8;
  k_paged_append<<<unsigned(blocks < most ? blocks : most), 256, 0, static_cast<cudaStream_t>(stream)>>>(p, a);
  REC_CHECK_CUDA(cudaGetLastError());
  return REC_OK;
}
