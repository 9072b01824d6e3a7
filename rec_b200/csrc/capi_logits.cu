// Per-row rules on a batch of logits: repetition, frequency and presence
// penalties by a row's own history, biases, an allow mask (rec_process_logits).
//
// One block per (row, chunk of the vocabulary).  Every thread first asks for
// its logits (16-byte pieces, all of them on their way before anything else);
// meanwhile the block marks, in one shared word per id, what the row's lists
// say of the ids of its chunk: bits 0-17 the id's count after the prompt, bits
// 18-30 one more than the last bias entry that names it, bit 31 whether the
// history has it at all.  A piece whose words are all 0 is copied, with the
// masked ids replaced; the others go through fp32.  The lists are read once
// per chunk (from L2 after the first), so the chunk is the largest that keeps
// the SMs busy, up to 8,192 ids (32 KB of words, 4 blocks an SM).
#include "capi_common.h"
#include "common.cuh"

using namespace rec;

namespace {

constexpr int kThreads = 512;
constexpr int kMaxChunk = 8192;
constexpr int kMaxHistory = (1 << 18) - 1;
constexpr int kMaxBias = (1 << 13) - 2;

struct LogitArgs {
  const void* in;
  void* out;
  int64_t stride, out_stride;
  int V, chunk;
  RecLogitRules r;
};

template <int T>
struct LogitType {
  using raw = uint16_t;
  static constexpr uint16_t low = T == REC_T_BF16 ? 0xFF80 : 0xFC00;  // -inf
  static __device__ __forceinline__ float get(raw x) { return T == REC_T_BF16 ? bf(x) : hf(x); }
  static __device__ __forceinline__ raw put(float x) {
    return T == REC_T_BF16 ? to_bf(x) : __half_as_ushort(__float2half_rn(x));
  }
};
template <>
struct LogitType<REC_T_FP32> {
  using raw = uint32_t;
  static constexpr uint32_t low = 0xFF800000u;
  static __device__ __forceinline__ float get(raw x) { return __uint_as_float(x); }
  static __device__ __forceinline__ raw put(float x) { return __float_as_uint(x); }
};

struct RowRules {
  float rho, freq, pres;
  const float* bias;
};
// The penalties and the bias that an id's word w asks for.
__device__ __forceinline__ float apply(float x, unsigned w, const RowRules& r) {
  if (w >> 31) x = x < 0.0f ? __fmul_rn(x, r.rho) : __fdiv_rn(x, r.rho);
  const unsigned c = w & 0x3FFFFu;
  if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.freq, float(c))), r.pres);
  const unsigned m = (w >> 18) & 0x1FFFu;
  if (m) x = __fadd_rn(x, r.bias[m - 1]);
  return x;
}

template <int T>
__global__ void __launch_bounds__(kThreads) k_process_logits(const LogitArgs a) {
  using L = LogitType<T>;
  using raw = typename L::raw;
  constexpr int E = 16 / sizeof(raw);                 // ids of a piece
  constexpr int N = kMaxChunk / E / kThreads;         // pieces of a thread
  __shared__ __align__(16) unsigned word[kMaxChunk];
  const int b = blockIdx.y;
  const RecLogitRules& r = a.r;
  const raw* in = static_cast<const raw*>(a.in) + b * a.stride;
  raw* out = static_cast<raw*>(a.out) + b * a.out_stride;
  // ids before the first 16-byte boundary of the row; the chunks start there
  const int skew = int((reinterpret_cast<uintptr_t>(in) & 15u) / sizeof(raw));
  const bool wide = skew == int((reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(raw));
  const int first = blockIdx.x * a.chunk - (wide ? skew : 0);  // id of word 0; below 0 at most in the first piece
  const int n = min(a.chunk, a.V - first);
  if (n <= 0) return;
  uint4 x[N];
  if (wide) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = (k * kThreads + threadIdx.x) * E;
      if (i + E <= n && first + i >= 0) x[k] = __ldcs(reinterpret_cast<const uint4*>(in + first + i));
    }
  }
  for (int i = 4 * threadIdx.x; i < n; i += 4 * kThreads) *reinterpret_cast<uint4*>(&word[i]) = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  const RowRules rules = {r.repetition ? __ldg(r.repetition + b) : 1.0f, r.frequency ? __ldg(r.frequency + b) : 0.0f,
                          r.presence ? __ldg(r.presence + b) : 0.0f, r.bias_values + int64_t(b) * r.n_bias};
  if (r.n_bias) {
    for (int j = threadIdx.x; j < r.n_bias; j += kThreads) {
      const int id = __ldg(r.bias_ids + int64_t(b) * r.n_bias + j);
      if (id >= 0 && id < a.V && unsigned(id - first) < unsigned(n)) atomicMax(&word[id - first], unsigned(j + 1) << 18);
    }
    __syncthreads();
  }
  if (r.history_cap) {
    const int len = min(r.history_cap, r.history_len ? max(0, __ldg(r.history_len + b)) : r.history_cap);
    const int prompt = r.prompt_len ? __ldg(r.prompt_len + b) : 0;
    const int* hist = r.history + int64_t(b) * r.history_cap;
#pragma unroll 4
    for (int j = threadIdx.x; j < len; j += kThreads) {
      const int id = __ldg(hist + j);
      if (id < 0 || id >= a.V || unsigned(id - first) >= unsigned(n)) continue;
      if (j < prompt) {
        atomicOr(&word[id - first], 0x80000000u);
      } else if (!((atomicAdd(&word[id - first], 1u)) >> 31)) {
        atomicOr(&word[id - first], 0x80000000u);
      }
    }
    __syncthreads();
  }
  const uint32_t* allow = r.allow ? r.allow + b * r.allow_stride : nullptr;
  auto one = [&](int i) {  // id first + i on its own
    const int id = first + i;
    if (id < 0) return;
    raw y = in[id];
    const unsigned w = word[i];
    if (w) y = L::put(apply(L::get(y), w, rules));
    if (allow && !((__ldg(allow + (id >> 5)) >> (id & 31)) & 1u)) y = L::low;
    out[id] = y;
  };
  if (!wide) {
    for (int i = threadIdx.x; i < n; i += kThreads) one(i);
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = (k * kThreads + threadIdx.x) * E;
    if (i >= n) break;
    if (i + E > n || first + i < 0) {
      for (int e = 0; e < E && i + e < n; ++e) one(i + e);
      continue;
    }
    unsigned w[E], any = 0u;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(&word[i + e]);
      w[e] = v.x, w[e + 1] = v.y, w[e + 2] = v.z, w[e + 3] = v.w;
      any |= v.x | v.y | v.z | v.w;
    }
    unsigned bits = (1u << E) - 1u;
    if (allow) {
      const int id = first + i, q = id >> 5, s = id & 31;
      const uint32_t lo = __ldg(allow + q), hi = s + E > 32 ? __ldg(allow + q + 1) : 0u;
      bits &= __funnelshift_r(lo, hi, s);
    }
    if (any || bits != (1u << E) - 1u) {
      raw y[E];
      *reinterpret_cast<uint4*>(y) = x[k];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (w[e]) y[e] = L::put(apply(L::get(y[e]), w[e], rules));
        if (!((bits >> e) & 1u)) y[e] = L::low;
      }
      x[k] = *reinterpret_cast<uint4*>(y);
    }
    __stcs(reinterpret_cast<uint4*>(out + first + i), x[k]);
  }
}

template <int T>
void launch(const LogitArgs& a, int batch, cudaStream_t st) {
  constexpr int E = 16 / int(sizeof(typename LogitType<T>::raw));
  const int64_t span = int64_t(a.V) + E - 1;  // with the row's skew
  k_process_logits<T><<<dim3(unsigned((span + a.chunk - 1) / a.chunk), batch), kThreads, 0, st>>>(a);
}

}  // namespace

REC_API int rec_process_logits(const void* logits, int64_t stride, void* logits_out, int64_t out_stride, int32_t dtype,
                               int32_t batch, int32_t vocab, const RecLogitRules* rules, void* stream) {
  REC_CHECK_ARG(logits && logits_out && rules, "rec_process_logits: null pointer");
  REC_CHECK_ARG(dtype == REC_T_BF16 || dtype == REC_T_FP16 || dtype == REC_T_FP32,
                "rec_process_logits: logits must be bf16, fp16 or fp32");
  const unsigned item = dtype == REC_T_FP32 ? 4 : 2;
  REC_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % item == 0 && reinterpret_cast<uintptr_t>(logits_out) % item == 0,
                "rec_process_logits: logits not aligned to their type");
  REC_CHECK_ARG(batch >= 1 && batch <= 4096, "rec_process_logits: batch %d outside 1..4096", batch);
  REC_CHECK_ARG(vocab >= 1 && vocab <= (1 << 24), "rec_process_logits: vocab %d outside 1..%d", vocab, 1 << 24);
  REC_CHECK_ARG(stride >= vocab && out_stride >= vocab, "rec_process_logits: row stride below vocab");
  const RecLogitRules& r = *rules;
  REC_CHECK_ARG(r.history_cap >= 0 && r.history_cap <= kMaxHistory && (r.history_cap == 0 || r.history),
                "rec_process_logits: history of %d ids (at most %d)", r.history_cap, kMaxHistory);
  REC_CHECK_ARG(r.n_bias >= 0 && r.n_bias <= kMaxBias && (r.n_bias == 0 || (r.bias_ids && r.bias_values)),
                "rec_process_logits: %d bias entries (at most %d)", r.n_bias, kMaxBias);
  REC_CHECK_ARG(!r.allow || r.allow_stride >= (vocab + 31) / 32, "rec_process_logits: allow rows too short");
  LogitArgs a = {logits, logits_out, stride, out_stride, vocab, kMaxChunk, r};
  // small batches: chunks of at least 1,024 ids until every SM has a block
  while (a.chunk > 1024 && int64_t(batch) * ((vocab + a.chunk - 1) / a.chunk) < sm_count()) a.chunk /= 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == REC_T_FP32) launch<REC_T_FP32>(a, batch, st);
  else if (dtype == REC_T_BF16) launch<REC_T_BF16>(a, batch, st);
  else launch<REC_T_FP16>(a, batch, st);
  REC_CHECK_CUDA(cudaGetLastError());
  return REC_OK;
}
