// Eviction from a paged cache by accumulated attention weight.
//
// Two kernels, both bound by latency and by the scattered rows' sectors.  The
// first selects: a cluster of 1 to 8 blocks per (session, kv head) holds the
// slots' rank keys in shared memory, finds the budget-th largest by up to
// three radix passes (11, 11 and 10 bits; the blocks' histograms meet in
// distributed shared memory; the passes end once every key that begins with
// the bits found stays), and lists the evicted slots below the budget and the
// kept slots at or above it, each in slot order.  32 rows of 4,352 slots take
// 14 us, of them 2.5 for the lengths, the table and the weights one after
// another, 4 for the three passes that weights with ties need; 32 rows of up
// to 65,536 slots 29 us.  The second kernel moves the r-th
// kept row to the r-th hole: lane m of a warp finds the places of move m and
// moves its scales, weight and position, then the warp moves the rows in
// 16-byte pieces, four on their way per lane.  Only holes are filled, so a cut
// of a few tokens moves a few rows; sources are at or above the budget and
// places below it, so no move reads what another wrote.
#include <limits.h>

#include "cluster.cuh"
#include "paged.cuh"

using namespace rec;

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kKeysInShared = 40960;  // of one block: 160 KB
constexpr int kMaxCluster = 8;

struct EvictArgs {
  const int* lengths;
  int* lengths_out;
  int budget;
  const float* w_in;
  float* w_out;
  const int* p_in;
  int* p_out;
  const int* keep_from;
  int keep_below;
  int *holes, *highs;   // [rows][cap] slots
  int* counts;          // [rows]
  int cap;
  uint32_t* keys;       // [rows][slots] when a block's keys exceed its shared memory, or NULL
  int cluster;
  int four;             // weights and positions can be read four slots at a time
  int* status;
};

struct SelectSmem {
  unsigned hist[3][kBins];  // read by the cluster's other blocks
  int scan[kWarps], scan2[kWarps];
  int pub[3];               // ties, holes, survivors of this block
  int digit[3], want[3], whole[3];
};

// Ascending in the rank order: 0 for NaN, ..., 0xFFFFFFFF protected.
__device__ __forceinline__ uint32_t rank_key(float w, bool keep) {
  if (keep) return 0xFFFFFFFFu;
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(__fadd_rn(w, 0.0f));  // -0 ranks as +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);       // +inf: 0xFF800000
}

// One more in bin d[k] for every lane and k with on[k]; together where the
// whole warp has one bin (weights that are all equal).
template <int N>
__device__ __forceinline__ void count_digits(unsigned* hist, const unsigned (&d)[N], const bool (&on)[N]) {
  unsigned lo = 0xFFFFFFFFu, hi = 0u, n = 0u;
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (on[k]) {
      lo = min(lo, d[k]);
      hi = max(hi, d[k]);
      ++n;
    }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lo == hi) {
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) atomicAdd(&hist[lo], n);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (on[k]) atomicAdd(&hist[d[k]], 1u);
  }
}

// Exclusive prefix of the warps' values; all is the block's sum.
__device__ __forceinline__ int warps_before(int v, int* scan, int& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) scan[warp] = v;
  __syncthreads();
  int x = scan[lane];
  all = __reduce_add_sync(0xffffffffu, x);
  x = lane < warp ? x : 0;
  return __reduce_add_sync(0xffffffffu, x);
}

// SHARED: the block's keys fit its shared memory.
template <bool SHARED>
__global__ void __launch_bounds__(kThreads) k_evict_select(const PagedView p, const EvictArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SelectSmem& sm = *reinterpret_cast<SelectSmem*>(smem_raw);
  auto sync = [&] {  // of the cluster; a block alone saves about 1,100 cycles a time
    if (a.cluster == 1) __syncthreads(); else cluster_sync_all();
  };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x / a.cluster, rank = int(cluster_rank()), b = row / p.hkv, h = row - b * p.hkv;
  int L = a.lengths[b];
  if (L < 0 || L > p.slots) {
    if (threadIdx.x == 0) report(a.status, kStatusBadPage);
    L = L < 0 ? 0 : int(p.slots);
  }
  const int budget = a.budget, kept = min(L, budget);
  // slots that stay below the budget are copied when the outputs are other tensors; a hole's copy is
  // overwritten by its move
  const bool copies = a.w_out != a.w_in || a.p_out != a.p_in;
  auto copy_slot = [&](int64_t at, int t, float w, int pos) {
    if (t >= kept) return;
    if (a.w_out != a.w_in) a.w_out[at] = w;
    if (a.p_out && a.p_out != a.p_in) a.p_out[at] = pos;
  };
  if (L <= budget || budget == 0) {  // the same for the whole cluster
    if (rank == 0 && threadIdx.x == 0) a.counts[row] = 0;
    if (copies)
      for (int t = rank * kThreads + threadIdx.x; t < kept; t += a.cluster * kThreads) {
        int off;
        const int page = slot_page(p, b, t, off);
        if (page < 0) continue;
        const int64_t at = slot_index(p, page, h, off);
        copy_slot(at, t, a.w_in[at], a.p_in ? a.p_in[at] : t);
      }
    return;
  }
  // this block's slots: [s0, s0 + n)
  const int slice = ((L + a.cluster - 1) / a.cluster + 31) & ~31;
  const int s0 = min(L, rank * slice), n = min(L, s0 + slice) - s0;
  uint32_t* keys = SHARED ? reinterpret_cast<uint32_t*>(smem_raw + sizeof(SelectSmem))
                          : a.keys + int64_t(row) * p.slots + s0;
  const int from = a.keep_from ? a.keep_from[b] : INT_MAX;
  // 8 slots of a thread on their way at once: two pieces of four, where a piece never crosses a page
  // (32 rows of 65,536 slots: 63.5 us for the call with single loads, 55 with pieces)
  auto slot_of = [&](int i0, int k) {
    return i0 + (a.four ? 4 * ((k >> 2) * kThreads + int(threadIdx.x)) + (k & 3) : k * kThreads + int(threadIdx.x));
  };
  bool cleared = false;
  for (int i0 = 0; i0 < n; i0 += 8 * kThreads) {
    int64_t at[8];
    float w[8];
    int pos[8];
    auto place = [&](int i) {
      int off;
      const int page = slot_page(p, b, s0 + i, off);
      if (page < 0) report(a.status, kStatusBadPage);
      return page < 0 ? int64_t(-1) : slot_index(p, page, h, off);
    };
    if (a.four) {
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        const int i = slot_of(i0, k);
        at[k] = i < n ? place(i) : -1;
#pragma unroll
        for (int e = 1; e < 4; ++e) at[k + e] = at[k] < 0 ? -1 : at[k] + e;
      }
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        int4 y = make_int4(s0 + slot_of(i0, k), s0 + slot_of(i0, k + 1), s0 + slot_of(i0, k + 2), s0 + slot_of(i0, k + 3));
        if (at[k] >= 0) {
          x = *reinterpret_cast<const float4*>(a.w_in + at[k]);
          if (a.p_in) y = *reinterpret_cast<const int4*>(a.p_in + at[k]);
        }
        w[k] = x.x, w[k + 1] = x.y, w[k + 2] = x.z, w[k + 3] = x.w;
        pos[k] = y.x, pos[k + 1] = y.y, pos[k + 2] = y.z, pos[k + 3] = y.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) at[k] = slot_of(i0, k) < n ? place(slot_of(i0, k)) : -1;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        w[k] = at[k] >= 0 ? a.w_in[at[k]] : 0.0f;
        pos[k] = at[k] >= 0 && a.p_in ? a.p_in[at[k]] : s0 + slot_of(i0, k);
      }
    }
    if (!cleared) {  // while the first loads are on their way
      for (int i = threadIdx.x; i < 3 * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(sm.hist)[i] = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
      cleared = true;
    }
    unsigned d[8];
    bool in[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = slot_of(i0, k);
      uint32_t key = 0u;  // also of a slot whose page is bad
      in[k] = i < n;
      if (in[k] && at[k] >= 0) {
        key = rank_key(w[k], pos[k] >= from || pos[k] < a.keep_below);
        if (copies) copy_slot(at[k], s0 + i, w[k], pos[k]);
      }
      if (in[k]) keys[i] = key;
      d[k] = key >> 21;
    }
    count_digits(sm.hist[0], d, in);
  }
  if (n == 0) {  // a cluster's last blocks may have no slots
    for (int i = threadIdx.x; i < 3 * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(sm.hist)[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
  }
  // the budget-th largest key's leading bits T, and how many of the keys that begin with them stay; once
  // all of those do, the bits after them decide nothing (for weights that differ, mostly after 22 bits)
  uint32_t T = 0;
  int want = budget, shift = 21;
  bool whole = false;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const unsigned bins = pass == 2 ? 1024u : 2048u;
    if (pass > 0)
      for (int i0 = 0; i0 < n; i0 += 4 * kThreads) {
        unsigned d[4];
        bool on[4];
        const int above = pass == 1 ? 21 : 10;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = i0 + k * kThreads + int(threadIdx.x);
          d[k] = i < n ? keys[i] : 0u;
          on[k] = i < n && (d[k] >> above) == T;
          d[k] = (d[k] >> shift) & (bins - 1);
        }
        if (__any_sync(0xffffffffu, on[0] || on[1] || on[2] || on[3])) count_digits(sm.hist[pass], d, on);
      }
    sync();
    // thread i sums bins 2(1023 - i) + 1 and 2(1023 - i): descending order
    const int d = 2 * (kThreads - 1 - int(threadIdx.x));
    int c1 = 0, c0 = 0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r)
      if (r < a.cluster) {
        const uint2 c = *reinterpret_cast<const uint2*>(peer(&sm.hist[pass][d], r));
        c0 += int(c.x);
        c1 += int(c.y);
      }
    int x = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    int all;
    const int before = warps_before(__shfl_sync(0xffffffffu, x, 31), sm.scan, all) + x - c0 - c1;
    if (before < want && want <= before + c0 + c1) {
      const bool upper = want <= before + c1;
      const int rest = want - before - (upper ? 0 : c1);
      sm.digit[pass] = upper ? d + 1 : d;
      sm.want[pass] = rest;
      sm.whole[pass] = rest == (upper ? c1 : c0);
    }
    __syncthreads();
    T = (T << (pass == 2 ? 10 : 11)) | uint32_t(sm.digit[pass]);
    want = sm.want[pass];
    whole = sm.whole[pass];
    if (whole) break;  // the same in every block
  }
  // a thread's slots are contiguous, so ranks in slot order are prefix counts; an odd number of them, so
  // that the threads' keys lie in different banks
  const int span = ((n + kThreads - 1) / kThreads) | 1;
  const int i_lo = min(n, int(threadIdx.x) * span), i_hi = min(n, i_lo + span);
  auto lanes_before = [&](int v, int& sum) {
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    sum = __shfl_sync(0xffffffffu, x, 31);
    return x - v;
  };
  // lane r of every warp reads block r's count
  auto of_peers = [&](int k, int& before) {
    const int x = lane < a.cluster ? *peer(&sm.pub[k], lane) : 0;
    before += __reduce_add_sync(0xffffffffu, lane < rank ? x : 0);
    return __reduce_add_sync(0xffffffffu, x);
  };
  int all, sum, tie0 = 0;
  if (!whole) {
    int ties = 0;
    for (int i = i_lo; i < i_hi; ++i) ties += keys[i] == T;  // all 32 bits here
    tie0 = lanes_before(ties, sum);
    tie0 += warps_before(sum, sm.scan, all);
    if (threadIdx.x == 0) sm.pub[0] = all;
    sync();
    of_peers(0, tie0);
  } else {
    want = INT_MAX;
  }
  auto each = [&](auto&& hole, auto&& high) {
    int tie = tie0;
    for (int i = i_lo; i < i_hi; ++i) {
      const uint32_t key = keys[i] >> shift;
      const bool keep = key > T || (key == T && tie++ < want);
      const int t = s0 + i;
      if (!keep && t < budget) hole(t);
      if (keep && t >= budget) high(t);
    }
  };
  int holes = 0, highs = 0;
  each([&](int) { ++holes; }, [&](int) { ++highs; });
  int high_at = lanes_before(highs, sum);
  if (lane == 0) sm.scan2[warp] = sum;
  int hole_at = lanes_before(holes, sum);
  hole_at += warps_before(sum, sm.scan, all);  // its barrier is also that of scan2
  if (threadIdx.x == 0) sm.pub[1] = all;
  const int other = sm.scan2[lane];
  high_at += __reduce_add_sync(0xffffffffu, lane < warp ? other : 0);
  all = __reduce_add_sync(0xffffffffu, other);
  if (threadIdx.x == 0) sm.pub[2] = all;
  sync();
  const int moves = of_peers(1, hole_at);
  of_peers(2, high_at);
  if (rank == 0 && threadIdx.x == 0) a.counts[row] = moves;
  int* hole_list = a.holes + int64_t(row) * a.cap;
  int* high_list = a.highs + int64_t(row) * a.cap;
  each([&](int t) { hole_list[hole_at++] = t; }, [&](int t) { high_list[high_at++] = t; });
  sync();  // a block's counts stay readable until every block has them
}

constexpr int kMoveThreads = 256;

// A warp takes M moves at a time.
template <int M>
__global__ void __launch_bounds__(kMoveThreads) k_evict_move(const PagedView p, const EvictArgs a, const FastDiv per) {
  grid_wait();  // launched once the selection's last block has left
  const int row = blockIdx.y, b = row / p.hkv, h = row - b * p.hkv, lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) {
    const int64_t L = max(0, a.lengths[b]);
    a.lengths_out[b] = int(min(min(L, p.slots), int64_t(a.budget)));
  }
  const int moves = a.counts[row];
  const int* hole_list = a.holes + int64_t(row) * a.cap;
  const int* high_list = a.highs + int64_t(row) * a.cap;
  const int nk = p.d * p.k_bits / 128, groups = p.k_bits == 16 ? 0 : p.d / 64;
  for (int m0 = (blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5)) * M; m0 < moves;
       m0 += gridDim.x * (kMoveThreads / 32) * M) {
    const int m = m0 + lane;
    int page_to = -1, off_to = 0, page_from = -1, off_from = 0;
    if (lane < M && m < moves) {
      const int to = hole_list[m], from = high_list[m];
      page_to = slot_page(p, b, to, off_to);
      page_from = slot_page(p, b, from, off_from);
      if (page_from < 0) page_to = -1;
      if (page_to >= 0) {
        const int64_t dst = slot_index(p, page_to, h, off_to), src = slot_index(p, page_from, h, off_from);
        const float w = a.w_in[src];
        const int pos = a.p_in ? a.p_in[src] : from;
        if (groups) {
          const size_t kd = scale_at(p.ks, page_to, h, off_to), kf = scale_at(p.ks, page_from, h, off_from);
          const size_t vd = scale_at(p.vs, page_to, h, off_to), vf = scale_at(p.vs, page_from, h, off_from);
          auto move4 = [&](auto* ks, auto* kb, auto* vs, auto* vb) {
            const auto x = ks[0], y = kb[0];
            const auto z = vs[0], u = vb[0];
            using T = decltype(ks);
            *reinterpret_cast<T>(p.ks.s + kd) = x;
            *reinterpret_cast<T>(p.ks.b + kd) = y;
            *reinterpret_cast<T>(p.vs.s + vd) = z;
            *reinterpret_cast<T>(p.vs.b + vd) = u;
          };
          if (groups == 1) move4(p.ks.s + kf, p.ks.b + kf, p.vs.s + vf, p.vs.b + vf);
          else if (groups == 2)
            move4(reinterpret_cast<uint32_t*>(p.ks.s + kf), reinterpret_cast<uint32_t*>(p.ks.b + kf),
                  reinterpret_cast<uint32_t*>(p.vs.s + vf), reinterpret_cast<uint32_t*>(p.vs.b + vf));
          else
            move4(reinterpret_cast<uint2*>(p.ks.s + kf), reinterpret_cast<uint2*>(p.ks.b + kf),
                  reinterpret_cast<uint2*>(p.vs.s + vf), reinterpret_cast<uint2*>(p.vs.b + vf));
        }
        a.w_out[dst] = w;
        if (a.p_out) a.p_out[dst] = pos;
      }
    }
    // the rows' pieces: K's, then V's
    const uint32_t k_to = page_to * p.k.page + h * p.k.head + off_to * p.k.row;
    const uint32_t v_to = page_to * p.v.page + h * p.v.head + off_to * p.v.row;
    const uint32_t k_from = page_from * p.k.page + h * p.k.head + off_from * p.k.row;
    const uint32_t v_from = page_from * p.v.page + h * p.v.head + off_from * p.v.row;
    const int pieces = min(M, moves - m0) * int(per.d);
    constexpr int U = 4;
    for (int x0 = 0; x0 < pieces; x0 += 32 * U) {
      uint4 val[U];
      uint8_t* dst[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int x = x0 + 32 * i + lane;
        const int mm = min(int(fdiv(x, per)), M - 1), e = x - int(fdiv(x, per)) * int(per.d);
        const bool there = __shfl_sync(0xffffffffu, page_to, mm) >= 0 && x < pieces;
        const uint32_t kt = __shfl_sync(0xffffffffu, k_to, mm), kf = __shfl_sync(0xffffffffu, k_from, mm);
        const uint32_t vt = __shfl_sync(0xffffffffu, v_to, mm), vf = __shfl_sync(0xffffffffu, v_from, mm);
        const bool is_k = e < nk;
        const size_t piece = size_t(is_k ? e : e - nk);
        dst[i] = there ? (is_k ? p.k.base : p.v.base) + ((size_t(is_k ? kt : vt) + piece) << 4) : nullptr;
        if (there)
          val[i] = __ldcs(reinterpret_cast<const uint4*>((is_k ? p.k.base : p.v.base) + ((size_t(is_k ? kf : vf) + piece) << 4)));
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (dst[i]) *reinterpret_cast<uint4*>(dst[i]) = val[i];
    }
  }
}

struct EvictLayout {
  int cluster, cap;
  bool shared;  // the keys fit shared memory
  size_t holes, highs, counts, keys, total;
};
EvictLayout evict_layout(int64_t slots, int batch, int hkv, int budget) {
  EvictLayout l;
  const int64_t rows = int64_t(batch) * hkv;
  auto slice = [&](int c) { return ((slots + c - 1) / c + 31) / 32 * 32; };
  // more blocks per row while a block has more than 4,096 keys and every block has an SM (one block
  // fills it: 8 sessions x 4 heads of 65,536 slots take 47 us in clusters of 4, 87 us in two waves of
  // clusters of 8; of 4,352 slots 16.7 us in clusters of 2, 17.2 alone, 18.9 in clusters of 4), or while
  // the keys do not fit
  l.cluster = 1;
  while (l.cluster < kMaxCluster && (slice(l.cluster) > kKeysInShared ||
                                     (slice(l.cluster) > 4096 && rows * l.cluster * 2 <= sm_count())))
    l.cluster *= 2;
  l.shared = slice(l.cluster) <= kKeysInShared;
  l.cap = int(slots < budget ? slots : budget);
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  l.holes = 0;
  l.highs = up(size_t(rows) * l.cap * 4);
  l.counts = 2 * l.highs;
  l.keys = l.counts + up(size_t(rows) * 4);
  l.total = l.keys + (l.shared ? 0 : up(size_t(rows) * size_t(slots) * 4));
  return l;
}

}  // namespace

REC_API size_t rec_paged_evict_workspace_bytes(const RecPagedKV* kv, const RecPagedTable* table, int32_t budget) {
  if (!kv || !table || budget < 0 || kv->n_kv_heads < 1 || kv->page_size < 1 || table->batch < 1 || table->width < 1)
    return 0;
  return evict_layout(int64_t(table->width) * kv->page_size, table->batch, kv->n_kv_heads, budget).total;
}

REC_API int rec_paged_evict(const RecPagedKV* kv, const RecPagedTable* table, const RecPagedEvict* evict,
                            void* workspace, size_t workspace_bytes, int32_t* status_dev, void* stream) {
  PagedView p;
  const int rc = paged_view(kv, table, "rec_paged_evict", &p);
  if (rc) return rc;
  REC_CHECK_ARG(evict && evict->lengths && evict->lengths_out && evict->weights_in && evict->weights_out,
                "rec_paged_evict: null lengths or weights");
  REC_CHECK_ARG(!evict->positions_in || evict->positions_out,
                "rec_paged_evict: positions_in without positions_out");
  REC_CHECK_ARG(evict->budget >= 0 && evict->keep_below >= 0, "rec_paged_evict: negative budget or keep_below");
  const EvictLayout l = evict_layout(p.slots, p.batch, p.hkv, evict->budget);
  REC_CHECK_ARG(workspace && workspace_bytes >= l.total && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0,
                "rec_paged_evict: workspace must be 256-byte aligned and hold %zu bytes", l.total);
  const int rows = p.batch * p.hkv;  // <= 4096 * 1024
  REC_CHECK_ARG(rows <= 65535, "rec_paged_evict: %d sessions times kv heads (at most 65,535)", rows);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  EvictArgs a = {};
  a.lengths = evict->lengths;
  a.lengths_out = evict->lengths_out;
  a.budget = evict->budget;
  a.w_in = evict->weights_in;
  a.w_out = evict->weights_out;
  a.p_in = evict->positions_in;
  a.p_out = evict->positions_out;
  a.keep_from = evict->keep_from;
  a.keep_below = evict->keep_below;
  a.holes = reinterpret_cast<int*>(ws + l.holes);
  a.highs = reinterpret_cast<int*>(ws + l.highs);
  a.counts = reinterpret_cast<int*>(ws + l.counts);
  a.cap = l.cap;
  a.keys = l.shared ? nullptr : reinterpret_cast<uint32_t*>(ws + l.keys);
  a.cluster = l.cluster;
  // a piece of four consecutive slots never crosses a page, and is aligned
  a.four = p.ps.d % 4 == 0 && aligned16(a.w_in) && (!a.p_in || aligned16(a.p_in));
  a.status = status_dev;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t slice = size_t((p.slots + l.cluster - 1) / l.cluster + 31) / 32 * 32;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * l.cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(SelectSmem) + (l.shared ? slice * 4 : 0);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {unsigned(l.cluster), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (l.shared) {
    REC_CHECK_CUDA(set_smem_limit(reinterpret_cast<const void*>(&k_evict_select<true>),
                                  sizeof(SelectSmem) + size_t(kKeysInShared) * 4));
    REC_CHECK_CUDA(cudaLaunchKernelEx(&cfg, k_evict_select<true>, p, a));
  } else {
    REC_CHECK_CUDA(cudaLaunchKernelEx(&cfg, k_evict_select<false>, p, a));
  }
  const FastDiv per = make_fastdiv(unsigned(p.d * (p.k_bits + p.v_bits) / 128));
  // moves of a row: no more than the budget, nor than the slots above it.  32 a warp; 8 where that
  // leaves SMs idle
  const int64_t most = p.slots > a.budget ? (p.slots - a.budget < l.cap ? p.slots - a.budget : l.cap) : 0;
  const int batch = most * rows >= int64_t(sm_count()) * 32 * 32 ? 32 : 8;
  const int64_t full = (most + 8 * batch - 1) / (8 * batch);  // blocks of 8 warps for a row's most moves
  int64_t x = (int64_t(sm_count()) * 8 + rows - 1) / rows;
  x = x < full ? x : full;
  cudaLaunchConfig_t mv = {};
  mv.gridDim = dim3(unsigned(x < 1 ? 1 : x), rows);
  mv.blockDim = dim3(kMoveThreads);
  mv.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  mv.attrs = attr;
  mv.numAttrs = 1;
  if (batch == 32) REC_CHECK_CUDA(cudaLaunchKernelEx(&mv, k_evict_move<32>, p, a, per));
  else REC_CHECK_CUDA(cudaLaunchKernelEx(&mv, k_evict_move<8>, p, a, per));
  return REC_OK;
}
