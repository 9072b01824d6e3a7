// Per-row rules on a batch of logits: repetition, frequency and presence
// penalties by a row's own history, biases, an allow mask (rec_process_logits).
//
// One block per (row, chunk of the vocabulary).  The logits stream through in
// 16-byte pieces, all of a thread's asked for before anything else, and only
// the mask touches them on the way; meanwhile the block marks, in one shared
// word per id, what the row's lists say of the ids of its chunk: bits 0-17 the
// id's count after the prompt, bits 18-30 one more than the last bias entry
// that names it, bit 31 whether the prompt has it.  The ids that get a
// word are listed once, and after the stream one thread each rewrites them: a
// history names a few percent of the ids, and looking for them in every piece
// would send every warp through the divisions.  The lists are read once per
// chunk (from L2 after the first), so the chunks are as few as fill whole
// waves of blocks, up to 18 ids a thread.  64 bf16 rows of 151,936 with
// histories of up to 4,096 take 16.8 us (41 MB: 2.4 TB/s; 6.5 us without any
// rule, 8 with the mask, 13.5 with the histories) in blocks of 1,024 threads,
// 19.5 in blocks of 512; one fp32 row 3.1 us in blocks of 512, 4.0 in blocks of
// 1,024.
#include "capi_common.h"
#include "common.cuh"

using namespace rec;

namespace {

constexpr int kIdsPerThread = 18;  // 6 bytes of shared memory each: 2,048 threads an SM
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
  const unsigned c = w & 0x3FFFFu;
  if (c || w >> 31) x = x < 0.0f ? __fmul_rn(x, r.rho) : __fdiv_rn(x, r.rho);
  if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.freq, float(c))), r.pres);
  const unsigned m = (w >> 18) & 0x1FFFu;
  if (m) x = __fadd_rn(x, r.bias[m - 1]);
  return x;
}

template <int T, int kThreads>
__global__ void __launch_bounds__(kThreads, 2048 / kThreads) k_process_logits(const LogitArgs a) {
  using L = LogitType<T>;
  using raw = typename L::raw;
  constexpr int E = 16 / sizeof(raw);                 // ids of a piece
  constexpr int N = (kIdsPerThread + E - 1) / E;      // pieces of a thread
  extern __shared__ __align__(16) unsigned word[];  // [chunk]
  uint16_t* listed = reinterpret_cast<uint16_t*>(word + a.chunk);
  __shared__ int n_listed;
  const int b = blockIdx.x;
  const RecLogitRules& r = a.r;
  const raw* in = static_cast<const raw*>(a.in) + b * a.stride;
  raw* out = static_cast<raw*>(a.out) + b * a.out_stride;
  // ids before the first 16-byte boundary of the row; the chunks start there
  const int skew = int((reinterpret_cast<uintptr_t>(in) & 15u) / sizeof(raw));
  const bool wide = skew == int((reinterpret_cast<uintptr_t>(out) & 15u) / sizeof(raw));
  const int first = blockIdx.y * a.chunk - (wide ? skew : 0);  // id of word 0; below 0 at most in the first piece
  const int n = min(a.chunk, a.V - first);
  if (n <= 0) return;
  const int len = min(r.history_cap, r.history_len ? max(0, __ldg(r.history_len + b)) : r.history_cap);
  const int prompt = r.prompt_len ? __ldg(r.prompt_len + b) : 0;
  uint4 x[N];
  if (wide) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = (k * kThreads + threadIdx.x) * E;
      if (i + E <= n && first + i >= 0) x[k] = __ldcs(reinterpret_cast<const uint4*>(in + first + i));
    }
  }
  const bool lists = r.n_bias || r.history_cap;
  if (lists) {
    if (threadIdx.x == 0) n_listed = 0;
    for (int i = 4 * threadIdx.x; i < n; i += 4 * kThreads)
      *reinterpret_cast<uint4*>(&word[i]) = make_uint4(0u, 0u, 0u, 0u);
  }
  const uint32_t* allow = r.allow ? r.allow + b * r.allow_stride : nullptr;
  auto allowed = [&](int id) { return !allow || ((__ldg(allow + (id >> 5)) >> (id & 31)) & 1u); };
  if (wide) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = (k * kThreads + threadIdx.x) * E;
      if (i >= n) break;
      if (i + E > n || first + i < 0) {  // the row's ends
        for (int e = 0; e < E && i + e < n; ++e)
          if (first + i + e >= 0) out[first + i + e] = allowed(first + i + e) ? in[first + i + e] : L::low;
        continue;
      }
      if (allow) {
        const int id = first + i, q = id >> 5, s = id & 31;
        const uint32_t lo = __ldg(allow + q), hi = s + E > 32 ? __ldg(allow + q + 1) : 0u;
        const unsigned bits = __funnelshift_r(lo, hi, s);
        uint32_t* y = reinterpret_cast<uint32_t*>(&x[k]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (E == 4) {
            y[j] = (bits >> j) & 1u ? y[j] : L::low;
          } else {  // all ones in the halves that stay
            const uint32_t m = ((bits >> (2 * j)) & 1u) * 0xFFFFu | ((bits >> (2 * j + 1)) & 1u) * 0xFFFF0000u;
            y[j] = (y[j] & m) | ((uint32_t(L::low) * 0x10001u) & ~m);
          }
        }
      }
      *reinterpret_cast<uint4*>(out + first + i) = x[k];
    }
  } else {
    for (int i = threadIdx.x; i < n; i += kThreads)
      if (first + i >= 0) out[first + i] = allowed(first + i) ? in[first + i] : L::low;
  }
  if (!lists) return;
  __syncthreads();
  auto list = [&](int i, unsigned before) {
    if (before == 0u) listed[atomicAdd(&n_listed, 1)] = uint16_t(i);
  };
  for (int j = threadIdx.x; j < r.n_bias; j += kThreads) {
    const int id = __ldg(r.bias_ids + int64_t(b) * r.n_bias + j);
    if (id < 0 || id >= a.V || unsigned(id - first) >= unsigned(n)) continue;
    // the last entry of an id, beside what the history has counted
    unsigned* at = &word[id - first];
    unsigned old = *at, was;
    do {
      was = old;
      if (((was >> 18) & 0x1FFFu) > unsigned(j)) break;
      old = atomicCAS(at, was, (was & ~(0x1FFFu << 18)) | unsigned(j + 1) << 18);
    } while (old != was);
    list(id - first, was);
  }
  if (r.history_cap) {
    const int* hist = r.history + int64_t(b) * r.history_cap;
    // the ids that count for this chunk: [max(first, 0), first + n), and first + n <= V
    const unsigned lo = unsigned(max(first, 0)), span = unsigned(first + n) - lo;
    constexpr int U = 4;
    for (int j0 = 0; j0 < len; j0 += U * kThreads) {
      unsigned id[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int j = j0 + k * kThreads + int(threadIdx.x);
        id[k] = j < len ? unsigned(__ldg(hist + j)) : 0xFFFFFFFFu;
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int j = j0 + k * kThreads + int(threadIdx.x);
        if (id[k] - lo >= span) continue;
        const int i = int(id[k]) - first;
        list(i, j < prompt ? atomicOr(&word[i], 0x80000000u) : atomicAdd(&word[i], 1u));
      }
    }
  }
  __syncthreads();
  const RowRules rules = {r.repetition ? __ldg(r.repetition + b) : 1.0f, r.frequency ? __ldg(r.frequency + b) : 0.0f,
                          r.presence ? __ldg(r.presence + b) : 0.0f, r.bias_values + int64_t(b) * r.n_bias};
  for (int k = threadIdx.x; k < n_listed; k += kThreads) {
    const int i = listed[k], id = first + i;
    // in place, a masked id reads as -inf here and stays that
    if (allowed(id)) out[id] = L::put(apply(L::get(in[id]), word[i], rules));
  }
}

template <int T, int kThreads>
cudaError_t launch(const LogitArgs& a, int batch, cudaStream_t st) {
  const void* f = reinterpret_cast<const void*>(&k_process_logits<T, kThreads>);
  const cudaError_t e = set_smem_limit(f, kIdsPerThread * kThreads * 6);
  if (e != cudaSuccess) return e;
  constexpr int E = 16 / int(sizeof(typename LogitType<T>::raw));
  const int64_t span = int64_t(a.V) + E - 1;  // with the row's skew
  k_process_logits<T, kThreads><<<dim3(batch, unsigned((span + a.chunk - 1) / a.chunk)), kThreads, a.chunk * 6, st>>>(a);
  return cudaGetLastError();
}

// Blocks of 512 threads where one wave of them covers the batch, of 1,024 for
// larger ones, so that a row's lists are read by half as many blocks.
template <int T>
cudaError_t launch(LogitArgs& a, int batch, cudaStream_t st) {
  const int64_t span = int64_t(a.V) + 7;
  const bool small = batch * ((span + kIdsPerThread * 512 - 1) / (kIdsPerThread * 512)) <= int64_t(sm_count()) * 4;
  // whole waves of blocks, and at least 1,024 ids a block
  const int64_t most = kIdsPerThread * (small ? 512 : 1024), wave = int64_t(sm_count()) * (small ? 4 : 2);
  const int64_t waves = (batch * ((span + most - 1) / most) + wave - 1) / wave;
  const int64_t chunks = wave * waves / batch;  // at least span / most of them
  const int64_t chunk = ((span + chunks - 1) / chunks + 15) / 16 * 16;
  a.chunk = int(chunk < 1024 ? 1024 : chunk < most ? chunk : most);
  return small ? launch<T, 512>(a, batch, st) : launch<T, 1024>(a, batch, st);
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
  REC_CHECK_ARG(!r.allow || r.allow_stride == 0 || r.allow_stride >= (vocab + 31) / 32, "rec_process_logits: allow rows too short");
  LogitArgs a = {logits, logits_out, stride, out_stride, vocab, 0, r};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == REC_T_FP32) REC_CHECK_CUDA(launch<REC_T_FP32>(a, batch, st));
  else if (dtype == REC_T_BF16) REC_CHECK_CUDA(launch<REC_T_BF16>(a, batch, st));
  else REC_CHECK_CUDA(launch<REC_T_FP16>(a, batch, st));
  return REC_OK;
}
