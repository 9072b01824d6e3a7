// Per-row rules on a batch of logits: repetition, frequency and presence
// penalties by a row's own history, biases, an allow mask (rec_process_logits).
//
// One block per (row, chunk of the vocabulary).  The block keeps one word per
// id of its chunk in shared memory: bits 0-17 the id's count after the prompt,
// bits 18-30 one more than the last bias entry that names it, bit 31 whether
// the history has it at all.  The row's lists are read once by every chunk;
// then the chunk's logits stream through, a word of 0 being a plain copy.
#include "capi_common.h"
#include "common.cuh"

using namespace rec;

namespace {

constexpr int kLogitThreads = 512;
constexpr int kLogitChunk = 8192;
constexpr int kLogitMaxHistory = (1 << 18) - 1;
constexpr int kLogitMaxBias = (1 << 13) - 2;

struct LogitArgs {
  const void* in;
  void* out;
  int64_t stride, out_stride;
  int V;
  RecLogitRules r;
};

template <int T>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
  if constexpr (T == REC_T_FP32) return static_cast<const float*>(p)[i];
  else if constexpr (T == REC_T_BF16) return bf(static_cast<const uint16_t*>(p)[i]);
  else return hf(static_cast<const uint16_t*>(p)[i]);
}
template <int T>
__device__ __forceinline__ void store_logit(void* p, int64_t i, float x) {
  if constexpr (T == REC_T_FP32) static_cast<float*>(p)[i] = x;
  else if constexpr (T == REC_T_BF16) static_cast<uint16_t*>(p)[i] = to_bf(x);
  else static_cast<uint16_t*>(p)[i] = __half_as_ushort(__float2half_rn(x));
}

template <int T>
__global__ void __launch_bounds__(kLogitThreads) k_process_logits(const LogitArgs a) {
  __shared__ unsigned word[kLogitChunk];
  const int b = blockIdx.y, i0 = blockIdx.x * kLogitChunk, n = min(kLogitChunk, a.V - i0);
  const RecLogitRules& r = a.r;
  for (int i = threadIdx.x; i < n; i += kLogitThreads) word[i] = 0u;
  __syncthreads();
  for (int j = threadIdx.x; j < r.n_bias; j += kLogitThreads) {
    const unsigned i = unsigned(r.bias_ids[int64_t(b) * r.n_bias + j]) - unsigned(i0);
    if (i < unsigned(n)) atomicMax(&word[i], unsigned(j + 1) << 18);
  }
  __syncthreads();
  const int len = min(r.history_cap, r.history_len ? max(0, r.history_len[b]) : r.history_cap);
  const int prompt = r.prompt_len ? r.prompt_len[b] : 0;
  for (int j = threadIdx.x; j < len; j += kLogitThreads) {
    const unsigned i = unsigned(r.history[int64_t(b) * r.history_cap + j]) - unsigned(i0);
    if (i >= unsigned(n)) continue;
    atomicOr(&word[i], 0x80000000u);
    if (j >= prompt) atomicAdd(&word[i], 1u);
  }
  __syncthreads();
  const float rho = r.repetition ? r.repetition[b] : 1.0f;
  const float freq = r.frequency ? r.frequency[b] : 0.0f;
  const float pres = r.presence ? r.presence[b] : 0.0f;
  for (int i = threadIdx.x; i < n; i += kLogitThreads) {
    const int id = i0 + i;
    float x = load_logit<T>(a.in, b * a.stride + id);
    const unsigned w = word[i];
    if (w) {
      if (w >> 31) x = x < 0.0f ? __fmul_rn(x, rho) : __fdiv_rn(x, rho);
      const unsigned c = w & 0x3FFFFu;
      if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, float(c))), pres);
      const unsigned m = (w >> 18) & 0x1FFFu;
      if (m) x = __fadd_rn(x, r.bias_values[int64_t(b) * r.n_bias + m - 1]);
    }
    if (r.allow && !((r.allow[b * r.allow_stride + (id >> 5)] >> (id & 31)) & 1u)) x = -INFINITY;
    store_logit<T>(a.out, b * a.out_stride + id, x);
  }
}

}  // namespace

REC_API int rec_process_logits(const void* logits, int64_t stride, void* logits_out, int64_t out_stride, int32_t dtype,
                               int32_t batch, int32_t vocab, const RecLogitRules* rules, void* stream) {
  REC_CHECK_ARG(logits && logits_out && rules, "rec_process_logits: null pointer");
  REC_CHECK_ARG(dtype == REC_T_BF16 || dtype == REC_T_FP16 || dtype == REC_T_FP32,
                "rec_process_logits: logits must be bf16, fp16 or fp32");
  REC_CHECK_ARG(batch >= 1 && batch <= 4096, "rec_process_logits: batch %d outside 1..4096", batch);
  REC_CHECK_ARG(vocab >= 1 && vocab <= (1 << 24), "rec_process_logits: vocab %d outside 1..%d", vocab, 1 << 24);
  REC_CHECK_ARG(stride >= vocab && out_stride >= vocab, "rec_process_logits: row stride below vocab");
  const RecLogitRules& r = *rules;
  REC_CHECK_ARG(r.history_cap >= 0 && r.history_cap <= kLogitMaxHistory && (r.history_cap == 0 || r.history),
                "rec_process_logits: history of %d ids (at most %d)", r.history_cap, kLogitMaxHistory);
  REC_CHECK_ARG(r.n_bias >= 0 && r.n_bias <= kLogitMaxBias && (r.n_bias == 0 || (r.bias_ids && r.bias_values)),
                "rec_process_logits: %d bias entries (at most %d)", r.n_bias, kLogitMaxBias);
  REC_CHECK_ARG(!r.allow || r.allow_stride >= (vocab + 31) / 32, "rec_process_logits: allow rows too short");
  LogitArgs a = {logits, logits_out, stride, out_stride, vocab, r};
  const dim3 grid((vocab + kLogitChunk - 1) / kLogitChunk, batch);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == REC_T_FP32) k_process_logits<REC_T_FP32><<<grid, kLogitThreads, 0, st>>>(a);
  else if (dtype == REC_T_BF16) k_process_logits<REC_T_BF16><<<grid, kLogitThreads, 0, st>>>(a);
  else k_process_logits<REC_T_FP16><<<grid, kLogitThreads, 0, st>>>(a);
  REC_CHECK_CUDA(cudaGetLastError());
  return REC_OK;
}
