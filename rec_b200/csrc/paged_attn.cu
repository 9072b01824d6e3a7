// Decode attention over a paged cache: one new token per session.
//
// One block per (query head, session): each warp takes every fourth slot, a
// slot's score by a butterfly over the lanes' dims, with a running maximum m,
// sum l and output acc (acc and l scaled by exp(m - m') when the maximum
// grows); the four warps' states join at the end.
#include "paged.cuh"

using namespace rec;

namespace {

constexpr int kWarps = 4;
constexpr int kMaxPerLane = 8;  // dims of a lane at head_dim 256

struct Args {
  const uint16_t* q;
  int64_t q_b, q_h;
  uint16_t* out;
  int64_t o_b, o_h;
  float* lse;
  const int* lengths;
  const uint16_t* sinks;
  int hq, G;
  float scale, cap;
  int window;
  const float* w_in;
  float* w_out;
  float decay;
  float* lse_ws;  // [batch][hq]
  int* status;
};

__device__ __forceinline__ float ld16(const uint16_t* p, int fp16) { return fp16 ? hf(*p) : bf(*p); }

// Dim d of a slot's row.
__device__ __forceinline__ float row_value(const uint8_t* row, const PagedScales& sc, size_t at, int bits, int fp16,
                                           int d) {
  if (bits == 16) return ld16(reinterpret_cast<const uint16_t*>(row) + d, fp16);
  const uint32_t w = reinterpret_cast<const uint32_t*>(row)[d * bits / 32];
  const float c = float((w >> (d * bits % 32)) & ((1u << bits) - 1u));
  return __fmaf_rn(c, bf(sc.s[at + d / 64]), bf(sc.b[at + d / 64]));
}

__device__ __forceinline__ int checked_length(const PagedView& p, const Args& a, int b) {
  const int L = a.lengths[b];
  if (L >= 0 && L <= p.slots) return L;
  report(a.status, kStatusBadPage);
  return L < 0 ? 0 : int(p.slots);
}

// The score of (query q, slot t); false when its page is bad.
__device__ __forceinline__ bool score(const PagedView& p, const Args& a, const float (&q)[kMaxPerLane], int page, int h,
                                      int off, float& s) {
  const int lane = threadIdx.x & 31;
  const uint8_t* row = row_ptr(p.k, page, h, off);
  const size_t at = scale_at(p.ks, page, h, off);
  float x = 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxPerLane; ++i)
    if (lane + 32 * i < p.d) x = __fmaf_rn(q[i], row_value(row, p.ks, at, p.k_bits, p.fp16, lane + 32 * i), x);
  s = bfly_sum(x) * a.scale;
  if (a.cap > 0.0f) s = a.cap * tanhf(s / a.cap);
  return true;
}

__global__ void __launch_bounds__(kWarps * 32) k_paged_attn(const PagedView p, const Args a) {
  __shared__ float sm_m[kWarps], sm_l[kWarps], sm_acc[kWarps][256];
  const int hq = blockIdx.x, b = blockIdx.y, h = hq / a.G, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int L = checked_length(p, a, b);
  const int lo = a.window > 0 ? max(0, L - a.window) : 0;
  float q[kMaxPerLane], acc[kMaxPerLane];
#pragma unroll
  for (int i = 0; i < kMaxPerLane; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < p.d ? ld16(a.q + b * a.q_b + hq * a.q_h + d, p.fp16) : 0.0f;
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int t = lo + warp; t < L; t += kWarps) {
    int off;
    const int page = slot_page(p, b, t, off);
    if (page < 0) {
      report(a.status, kStatusBadPage);
      continue;
    }
    float s;
    score(p, a, q, page, h, off, s);
    const float mn = fmaxf(m, s);
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float alpha = __expf(m - ref), w = __expf(s - ref);
    m = mn;
    l = l * alpha + w;
    const uint8_t* row = row_ptr(p.v, page, h, off);
    const size_t at = scale_at(p.vs, page, h, off);
#pragma unroll
    for (int i = 0; i < kMaxPerLane; ++i)
      if (lane + 32 * i < p.d)
        acc[i] = __fmaf_rn(w, row_value(row, p.vs, at, p.v_bits, p.fp16, lane + 32 * i), acc[i] * alpha);
  }
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < kMaxPerLane; ++i) sm_acc[warp][lane + 32 * i] = acc[i];
  __syncthreads();
  const float sink = a.sinks ? bf(a.sinks[hq]) : -INFINITY;
  float M = sink;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w]);
  const float ref = M == -INFINITY ? 0.0f : M;
  float total = __expf(sink - ref);
  for (int w = 0; w < kWarps; ++w) total += sm_l[w] * __expf(sm_m[w] - ref);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  for (int d = threadIdx.x; d < p.d; d += kWarps * 32) {
    float o = 0.0f;
    for (int w = 0; w < kWarps; ++w) o += sm_acc[w][d] * __expf(sm_m[w] - ref);
    o *= inv;
    a.out[b * a.o_b + hq * a.o_h + d] = p.fp16 ? __half_as_ushort(__float2half_rn(o)) : to_bf(o);
  }
  if (threadIdx.x == 0) {
    const float lse = total == 0.0f ? -INFINITY : ref + logf(total);
    if (a.lse) a.lse[b * a.hq + hq] = lse;
    a.lse_ws[b * a.hq + hq] = lse;
  }
}

// weights_out = decay * weights_in + the slot's weights summed over the kv
// head's query heads; one warp per slot.
__global__ void __launch_bounds__(kWarps * 32) k_paged_weights(const PagedView p, const Args a) {
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int L = checked_length(p, a, b);
  const int lo = a.window > 0 ? max(0, L - a.window) : 0;
  for (int t = blockIdx.z * kWarps + warp; t < L; t += gridDim.z * kWarps) {
    int off;
    const int page = slot_page(p, b, t, off);
    if (page < 0) continue;
    float w = 0.0f;
    for (int g = 0; g < a.G && t >= lo; ++g) {
      float q[kMaxPerLane], s;
#pragma unroll
      for (int i = 0; i < kMaxPerLane; ++i) {
        const int d = lane + 32 * i;
        q[i] = d < p.d ? ld16(a.q + b * a.q_b + (h * a.G + g) * a.q_h + d, p.fp16) : 0.0f;
      }
      score(p, a, q, page, h, off, s);
      w += __expf(s - a.lse_ws[b * a.hq + h * a.G + g]);
    }
    if (lane == 0) {
      const int64_t at = slot_index(p, page, h, off);
      a.w_out[at] = a.decay != 0.0f ? __fmaf_rn(a.decay, a.w_in[at], w) : w;
    }
  }
}

}  // namespace

REC_API size_t rec_paged_attn_workspace_bytes(const RecPagedKV* kv, const RecPagedTable* table, int32_t n_q_heads,
                                              int32_t weights, size_t* zeroed) {
  if (!kv || !table || n_q_heads < 1 || table->batch < 1) return 0;
  if (zeroed) *zeroed = 0;
  return (size_t(table->batch) * n_q_heads * 4 + 255) / 256 * 256;
}

REC_API int rec_paged_attn_decode(const RecPagedKV* kv, const RecPagedTable* table, const RecPagedAttn* attn,
                                  void* workspace, size_t workspace_bytes, int32_t* status_dev, void* stream) {
  PagedView p;
  const int rc = paged_view(kv, table, "rec_paged_attn_decode", &p);
  if (rc) return rc;
  REC_CHECK_ARG(attn && attn->q && attn->out && attn->lengths, "rec_paged_attn_decode: null pointer");
  const RecPagedAttn& t = *attn;
  REC_CHECK_ARG(aligned16(t.q) && aligned16(t.out) && t.q_batch_stride % 8 == 0 && t.q_head_stride % 8 == 0 &&
                    t.out_batch_stride % 8 == 0 && t.out_head_stride % 8 == 0,
                "rec_paged_attn_decode: q and out rows must be 16-byte aligned");
  REC_CHECK_ARG(t.n_q_heads >= 1 && t.n_q_heads % p.hkv == 0 && t.n_q_heads <= 65536,
                "rec_paged_attn_decode: %d query heads over %d kv heads", t.n_q_heads, p.hkv);
  REC_CHECK_ARG(t.scale > 0.0f && t.scale < 1e30f && t.softcap >= 0.0f && t.softcap < 1e30f && t.window >= 0,
                "rec_paged_attn_decode: bad scale, softcap or window");
  REC_CHECK_ARG(!t.weights_out || t.decay == 0.0f || t.weights_in,
                "rec_paged_attn_decode: decay without weights_in");
  const size_t need = rec_paged_attn_workspace_bytes(kv, table, t.n_q_heads, t.weights_out != nullptr, nullptr);
  REC_CHECK_ARG(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
                "rec_paged_attn_decode: workspace must be 256-byte aligned and hold %zu bytes", need);
  Args a = {};
  a.q = static_cast<const uint16_t*>(t.q);
  a.q_b = t.q_batch_stride;
  a.q_h = t.q_head_stride;
  a.out = static_cast<uint16_t*>(t.out);
  a.o_b = t.out_batch_stride;
  a.o_h = t.out_head_stride;
  a.lse = t.lse;
  a.lengths = t.lengths;
  a.sinks = static_cast<const uint16_t*>(t.sinks);
  a.hq = t.n_q_heads;
  a.G = t.n_q_heads / p.hkv;
  a.scale = t.scale;
  a.cap = t.softcap;
  a.window = t.window;
  a.w_in = t.weights_in;
  a.w_out = t.weights_out;
  a.decay = t.decay;
  a.lse_ws = static_cast<float*>(workspace);
  a.status = status_dev;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  k_paged_attn<<<dim3(a.hq, p.batch), kWarps * 32, 0, st>>>(p, a);
  REC_CHECK_CUDA(cudaGetLastError());
  if (a.w_out) {
    k_paged_weights<<<dim3(p.hkv, p.batch, 32), kWarps * 32, 0, st>>>(p, a);
    REC_CHECK_CUDA(cudaGetLastError());
  }
  return REC_OK;
}
