// Paged decode attention: entry points, and the accumulation of the weights.
#include "paged_attn.cuh"

using namespace rec;

namespace rec {

PagedAttnShape paged_attn_shape(const PagedView& p, int group) {
  const int dp = p.d <= 64 ? 64 : p.d <= 128 ? 128 : 256;
  return {dp, group <= 8 || dp == 256 ? 8 : 16, 1};
}

}  // namespace rec

namespace {

constexpr int kWeightThreads = 256;

// weights_out = decay * weights_in + sum over the kv head's query heads of
// 2^(score - lse), from the scores the attention kernel left.  One thread per
// slot; units of 256 slots shared out as the attention's are.
__global__ void __launch_bounds__(kWeightThreads) k_paged_weights(const PagedView p, const PagedAttnArgs a) {
  extern __shared__ int plan[];
  __shared__ int scan[32];
  int* len = plan;
  int* pre = plan + p.batch;
  plan_units(p, a.lengths, nullptr, kWeightThreads, len, pre, scan,
             [](int L) { return max(1, (L + kWeightThreads - 1) / kWeightThreads); });
  // launched once the attention's last block has left; what it wrote is read by plain loads, which stay below
  grid_wait();
  const int64_t H = p.hkv, total = pre[p.batch] * H;
  for (int64_t u = blockIdx.x; u < total; u += gridDim.x) {
    const int b = unit_session(pre, p.batch, H, u);
    const int64_t rest = u - pre[b] * H;
    const int nb = pre[b + 1] - pre[b], h = int(rest / nb);
    const int t = int(rest % nb) * kWeightThreads + int(threadIdx.x), L = len[b];
    if (t >= L) continue;
    int off;
    const int page = slot_page(p, b, t, off);
    if (page < 0) {  // (below the window the attention has not looked)
      report(a.status, kStatusBadPage);
      continue;
    }
    float w = 0.0f;
    if (a.window <= 0 || t >= L - a.window) {
      const float* sc = a.scores + (int64_t(b * p.hkv + h) * a.score_len + t) * a.G;
      const float* ls = a.lse2 + b * a.hq + h * a.G;
      // the scores of a slot's heads lie together; four at a time where a row of them is aligned
      if (a.G % 4 == 0) {
        for (int g = 0; g < a.G; g += 4) {
          const float4 x = *reinterpret_cast<const float4*>(sc + g);
          w += ex2(x.x - ls[g]) + ex2(x.y - ls[g + 1]) + ex2(x.z - ls[g + 2]) + ex2(x.w - ls[g + 3]);
        }
      } else {
        for (int g = 0; g < a.G; ++g) w += ex2(sc[g] - ls[g]);
      }
    }
    const int64_t at = slot_index(p, page, h, off);
    a.w_out[at] = a.decay != 0.0f ? __fmaf_rn(a.decay, a.w_in[at], w) : w;
  }
}

struct Layout {
  size_t counters, part_ml, part_acc, lse2, scores, total;  // counters: the size of that buffer
};
Layout layout_of(const PagedView& p, int hq, bool weights) {
  const PagedAttnShape s = paged_attn_shape(p, hq / p.hkv);
  const int hb = (hq / p.hkv + s.hn - 1) / s.hn;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const size_t slots = size_t(2) * sm_count() * s.blocks;
  Layout l;
  l.counters = size_t(p.batch) * p.hkv * hb * 4;
  l.part_ml = 0;
  l.part_acc = l.part_ml + up(slots * s.hn * 8);
  l.lse2 = l.part_acc + up(slots * s.hn * s.dp * 4);
  l.scores = l.lse2 + (weights ? up(size_t(p.batch) * hq * 4) : 0);
  l.total = l.scores + (weights ? up(size_t(p.batch) * hq * size_t(p.slots) * 4) : 0);
  return l;
}

}  // namespace

REC_API size_t rec_paged_attn_workspace_bytes(const RecPagedKV* kv, const RecPagedTable* table, int32_t n_q_heads,
                                              int32_t weights, size_t* counter_bytes) {
  PagedView p;
  if (paged_view(kv, table, "rec_paged_attn_workspace_bytes", &p)) return 0;
  if (n_q_heads < 1 || n_q_heads % p.hkv) return 0;
  const Layout l = layout_of(p, n_q_heads, weights != 0);
  if (counter_bytes) *counter_bytes = l.counters;
  return l.total;
}

REC_API int rec_paged_attn_decode(const RecPagedKV* kv, const RecPagedTable* table, const RecPagedAttn* attn,
                                  void* workspace, size_t workspace_bytes, uint32_t* counters, size_t counter_bytes,
                                  int32_t* status_dev, void* stream) {
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
  // so that the units of all sessions (of 128 slots or more) fit 31 bits
  REC_CHECK_ARG(p.batch * p.slots <= int64_t(1) << 37, "rec_paged_attn_decode: a table of %lld slots", (long long)(p.batch * p.slots));
  const Layout l = layout_of(p, t.n_q_heads, t.weights_out != nullptr);
  REC_CHECK_ARG(workspace && workspace_bytes >= l.total && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
                "rec_paged_attn_decode: workspace must be 256-byte aligned and hold %zu bytes", l.total);
  REC_CHECK_ARG(counters && counter_bytes >= l.counters && (reinterpret_cast<uintptr_t>(counters) & 3u) == 0,
                "rec_paged_attn_decode: counters must be 4-byte aligned and hold %zu bytes", l.counters);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  PagedAttnArgs a = {};
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
  const PagedAttnShape s = paged_attn_shape(p, a.G);
  a.HB = (a.G + s.hn - 1) / s.hn;
  a.scale_log2 = t.scale * kLog2e;
  if (t.softcap > 0.0f) {
    a.cap_in = t.scale / t.softcap;
    a.cap_out = t.softcap * kLog2e;
  }
  a.window = t.window;
  a.counters = counters;
  a.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
  a.part_acc = reinterpret_cast<float*>(ws + l.part_acc);
  if (t.weights_out) {
    a.lse2 = reinterpret_cast<float*>(ws + l.lse2);
    a.scores = reinterpret_cast<float*>(ws + l.scores);
    a.score_len = p.slots;
  }
  a.w_in = t.weights_in;
  a.w_out = t.weights_out;
  a.decay = t.decay;
  a.status = status_dev;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sms = sm_count();
  if (p.k_bits == 16) REC_CHECK_CUDA(p.fp16 ? paged_attn_fp16(p, a, sms, st) : paged_attn_bf16(p, a, sms, st));
  else REC_CHECK_CUDA(p.k_bits == 8 ? paged_attn_codes8(p, a, sms, st) : paged_attn_codes4(p, a, sms, st));
  if (a.w_out) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(sms) * 8);
    cfg.blockDim = dim3(kWeightThreads);
    cfg.dynamicSmemBytes = size_t(2 * p.batch + 1) * sizeof(int);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    REC_CHECK_CUDA(cudaLaunchKernelEx(&cfg, k_paged_weights, p, a));
  }
  return REC_OK;
}
