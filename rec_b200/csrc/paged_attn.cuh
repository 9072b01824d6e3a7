// Decode attention over a paged cache: one new token per session, every
// session of its own length.
//
// Work.  The slots that a session attends are cut into units of UT =
// W * 16 * TT slots; the units of every (session, kv head, block of HN query
// heads) follow one another in one list that the grid shares out evenly, so
// neither a long session nor many short ones leave an SM idle.  A block walks
// its share segment by segment (a segment: its units of one (session, head));
// a segment that is not the whole list of its head leaves a partial state,
// and the last block to finish a head joins the partials in block order.  A
// join takes 2 to 3.5 us, as long as one or two units, so where every head can
// have a block of its own and none is longer than WHOLE units beyond an even
// share, a block takes a whole head.  One session with 4 kv heads, split and
// whole: 300 slots of bf16 9.4 and 8.1 us, 600 slots of 8-bit codes 10.6 and
// 10.1 (one more unit); 450 slots of fp16, 64 dims, 8.4 and 7.4 (two more).  A
// second unit more costs where a unit is long: 800 slots of 8-bit codes 10.9
// split, 12.1 whole (units of 384 slots), 300 of bf16, 256 dims, 11.3 and 11.9.
//
// Tile.  A warp folds 16 * TT slots at a time on the tensor cores
// (mma.m16n8k16), with the cache as the A operand so that 8 query heads fill
// the n side: S^T = K Q^T, then O^T += V^T P^T.  A product's k order is free
// as long as both sides agree, so every lane loads 16 bytes of a row straight
// into the registers that the MMA reads: no shared memory, no transposition
// for K, and one byte permutation per register for V (two slots of one dim
// into a pair).  K of the next tile is on its way while this tile's softmax
// and PV run, V while the next scores run; where every block has more than 16
// tiles a warp, 16-bit rows are also asked for in L2 a tile earlier (64 sessions
// up to 16K: 188 -> 181 us; over ten tiles a warp it costs more than it brings,
// 45.4 -> 47.5 us, and so it does for codes, whose widening takes as many
// instructions again).  All blocks or none: asking in long segments only
// starved the blocks with short ones (220 us), and without the next segment's
// first tiles nothing is gained.
// Loads on their way hold L1 space, so shared memory is kept small: 227 KB of
// it instead of 54 took the same case from 188 to 241 us.
//
// Softmax.  s in log2 units; a reference per head follows the running maximum
// when it is passed by more than 8 (bf16: p <= 256 until then) or 4 (fp16), so
// most tiles need no reduction over the warp and no rescaling.  p enters the
// PV product as two 16-bit numbers, high and low part: a relative 2^-16 for
// bf16.  fp16 ends at 2^-24, so there the reference lies 2^9 below the maximum:
// two parts keep 2^-22 of p, and no less than 2^-34 of the largest weight in
// the warp, where p against the maximum itself would lose every weight below
// 2^-25 of it whole.  The second MMA is free, the kernel is bound by the
// cache's bytes (64 sessions up to 8K of fp16: 105 us with either reference).
//
// Quantized rows.  score = sum_g scale_g (q . c_g) + bias_g sum(q_g) over the
// 64-dim groups, with the codes centred (c - 128 or c - 8: exact in fp16, and
// the bias term then cancels little); q enters as fp16 after a power of two
// that brings the head's largest value into [1, 2), so what fp16 loses is
// below 2^-25 of it.  PV: p * scale_g is the P operand of group g, in two fp16
// parts as above.  Its size is what has to fit fp16, so the reference follows
// the maximum of score + log2(largest |scale| of the slot): p itself is fp32
// and takes any unit, and a slot whose scale is large but whose weight is
// small costs the others nothing.  The warps' units meet again when a segment
// ends (each state brought to a sum in [1, 2)).  sum p * bias_g is added to the
// group's dims there, in fp32.  One fp16 part (2^-11 of a weight) would be 4 to
// 5 % faster (131,072 slots of 8 bits 42.9 against 44.9 us) and would move
// outputs by 7.5e-4 in the 2-norm.
#pragma once
#include "paged.cuh"

namespace rec {

struct PagedAttnArgs {
  const uint16_t* q;
  int64_t q_b, q_h;
  uint16_t* out;
  int64_t o_b, o_h;
  float* lse;
  const int* lengths;
  const uint16_t* sinks;
  int hq, G, HB;      // query heads, per kv head, blocks of HN of them
  float scale_log2;   // scale * log2(e)
  float cap_in;       // scale / cap
  float cap_out;      // cap * log2(e); 0: no cap
  int window;
  unsigned* counters; // [batch * hkv * HB], zero between calls
  float* part_acc;    // [2 * grid][HN][DP]
  float2* part_ml;    // [2 * grid][HN]
  float* scores;      // [batch * hkv][score_len][G] log2 units, or NULL
  int64_t score_len;
  float* lse2;        // [batch][hq] in log2 units (with scores)
  const float* w_in;
  float* w_out;
  float decay;
  int* status;
};

constexpr int kPagedMaxBatch = 4096;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
// The transpose of an 8x8 matrix of 16-bit values held as row lane/4,
// columns 2 (lane % 4) and the next.
__device__ __forceinline__ uint32_t trans8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// (lo, hi) as a pair of 16-bit values, and back.
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if constexpr (F16)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool F16>
__device__ __forceinline__ float2 unpack16(uint32_t v) {
  if constexpr (F16) return __half22float2(*reinterpret_cast<__half2*>(&v));
  else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// Centred fp16 pairs from codes: 0x6400 | n is 1024 + n in fp16.
__device__ __forceinline__ uint32_t nib_even(uint32_t y) {  // nibbles 0 and 4 of y, minus 8
  return hsub2((y & 0x000F000Fu) | 0x64006400u, 0x64086408u);
}
__device__ __forceinline__ uint32_t nib_odd(uint32_t y) {  // nibbles 1 and 5: 1024 + 16 n, times 1/16, minus 72
  return hfma2((y & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u);
}
template <int SEL>
__device__ __forceinline__ uint32_t byte_pair(uint32_t x) {  // two bytes of x, minus 128
  return hsub2(prmt(x, 0x64646464u, SEL), 0x64806480u);
}

template <int N>
__device__ __forceinline__ void ldg_words(uint32_t* r, const uint8_t* p) {
  if constexpr (N == 4)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "l"(p));
  else if constexpr (N == 2)
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
  else
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r[0]) : "l"(p));
}

// KB, VB: bits of the rows.  F16: fp16 MMAs (fp16 rows, or codes).  DP: the
// head dim's padded size (64, 128, 256).  NT: n tiles of 8 query heads.  TT:
// m tiles of 16 slots per warp and step.  W: warps of a block.  MINB: blocks
// of an SM.
template <int KB_, int VB_, bool F16_, int DP_, int NT_, int TT_, int W_, int MINB_>
struct PagedCfg {
  static constexpr int KB = KB_, VB = VB_, DP = DP_, NT = NT_, TT = TT_, W = W_, MINB = MINB_;
  static constexpr bool F16 = F16_, Q = KB_ != 16;
  static constexpr int HN = 8 * NT, NG = DP / 64, TS = 16 * TT, UT = W * TS;
  static constexpr int KW = KB == 16 ? DP / 8 : NG * (KB == 8 ? 4 : 2);  // words of a K row per lane
  static constexpr int VW = VB == 16 ? NG * 4 : NG * (VB == 8 ? 2 : 1);  // words of a V row per lane
  static constexpr int SW = (NG + 1) / 2;                                // words of a row's scales
  static constexpr int QP = DP + 32;                                     // pitch of a query in shared memory
  static constexpr int RP = DP + 4;                                      // pitch of a head's state there
  // The reference moves when a score passes the maximum by more than LAG, and then lies REF below it: fp16
  // MMAs take p from 2^9 (at the maximum) up to 2^14 (codes: p * scale, below 2^15), bf16 needs no such place.
  // (LAG 2 and REF 11 would gain two bits and cost codes 0.5 %.)
  static constexpr float LAG = F16 ? 4.0f : 8.0f, REF = F16 ? 9.0f : 0.0f;
  // Units beyond an even share up to which a block takes a whole head.
  static constexpr int WHOLE = TT == 2 || (!Q && DP == 256) ? 1 : 2;
};

template <class C>
struct PagedSmem {
  alignas(16) uint16_t q[C::HN][C::QP];
  float qsum[C::HN][C::NG];  // codes: sums of the scaled query over each group
  float qfac[C::HN];         // codes: the power of two back
  float m[C::W][C::HN], l[C::W][C::HN];
  float head_m[C::HN], head_l[C::HN];
  int scan[32];
  int last;
  int64_t per;  // units of a block's share
  alignas(16) float acc[C::W][C::HN][C::RP];  // joins: weights of the partials
  // then: int len[batch], pre[batch + 1]
};

// What a block knows of its current segment.
struct PagedSeg {
  int b, hh, h, L, lo;
  int ul, n, nb;  // first unit, units here, units of the head
};

template <class C>
struct PagedTile {
  uint32_t k[C::TT][2][C::KW], v[C::TT][4][C::VW];
  uint32_t ks[C::SW], kb[C::SW], vs[C::SW], vb[C::SW];  // codes: of the lane's own slot (0 past the end)
};

// Where a lane's slot of the coming tile is, in the pools' units.
struct PagedPlace {
  uint32_t k, v, ks, vs;
  uint32_t valid;  // one bit per slot of the tile, the same in every lane
};

template <int SW>
__device__ __forceinline__ float scale_of(const uint32_t (&w)[SW], int g) {
  return g & 1 ? __uint_as_float(w[g >> 1] & 0xFFFF0000u) : __uint_as_float(w[g >> 1] << 16);
}
// A slot's scales and biases; 0 when it is not there.
template <int NG, int SW>
__device__ __forceinline__ void load_scales(uint32_t (&s)[SW], uint32_t (&b)[SW], const PagedScales& p, uint32_t at,
                                            bool there) {
#pragma unroll
  for (int i = 0; i < SW; ++i) s[i] = b[i] = 0u;
  if (!there) return;
  if constexpr (NG == 1) {
    s[0] = __ldg(p.s + at);
    b[0] = __ldg(p.b + at);
  } else if constexpr (NG == 2) {
    s[0] = __ldg(reinterpret_cast<const unsigned*>(p.s + at));
    b[0] = __ldg(reinterpret_cast<const unsigned*>(p.b + at));
  } else {
    const uint2 x = __ldg(reinterpret_cast<const uint2*>(p.s + at)), y = __ldg(reinterpret_cast<const uint2*>(p.b + at));
    s[0] = x.x, s[1] = x.y, b[0] = y.x, b[1] = y.y;
  }
}
// The words of another lane's slot.
template <int SW>
__device__ __forceinline__ void from_lane(uint32_t (&d)[SW], const uint32_t (&w)[SW], int lane) {
#pragma unroll
  for (int i = 0; i < SW; ++i) d[i] = __shfl_sync(0xffffffffu, w[i], lane);
}

// Places of the TS slots from t0 of a segment (lane i: slot t0 + i % TS).
template <class C>
__device__ __forceinline__ void find_places(const PagedView& p, const PagedAttnArgs& a, const PagedSeg& s, int t0,
                                            PagedPlace& at) {
  const int lane = threadIdx.x & 31;
  const int t = t0 + (lane & (C::TS - 1));
  bool ok = t < s.L;
  int off = 0, page = 0;
  if (ok) {
    page = slot_page(p, s.b, t, off);
    if (page < 0) {
      report(a.status, kStatusBadPage);
      ok = false;
      page = off = 0;
    }
  }
  at.k = page * p.k.page + s.h * p.k.head + off * p.k.row;
  at.v = page * p.v.page + s.h * p.v.head + off * p.v.row;
  if constexpr (C::Q) {
    at.ks = page * p.ks.page + s.h * p.ks.head + off * p.ks.row;
    at.vs = page * p.vs.page + s.h * p.vs.head + off * p.vs.row;
  }
  at.valid = __ballot_sync(0xffffffffu, ok) & (C::TS == 32 ? 0xffffffffu : (1u << C::TS) - 1u);
}

// Asks for the rows of the tile from t0 in L2.
template <class C>
__device__ __forceinline__ void prefetch_tile(const PagedView& p, const PagedSeg& s, int t0) {
  const int lane = threadIdx.x & 31, part = lane / C::TS;  // 32 / TS lanes a slot, 128 bytes at a time
  const int t = t0 + (lane & (C::TS - 1));
  if (t >= s.L) return;
  int off;
  const int page = slot_page(p, s.b, t, off);
  if (page < 0) return;
  const uint8_t* k = row_ptr(p.k, page, s.h, off);
  const uint8_t* v = row_ptr(p.v, page, s.h, off);
#pragma unroll
  for (int o = 0; o < 2 * C::DP; o += 128 * (32 / C::TS)) {
    const int x = o + 128 * part;
    if (x < 2 * p.d) {
      asm volatile("prefetch.global.L2 [%0];" ::"l"(k + x));
      asm volatile("prefetch.global.L2 [%0];" ::"l"(v + x));
    }
  }
}

template <class C>
__device__ __forceinline__ void load_k(const PagedView& p, const PagedPlace& at, PagedTile<C>& f) {
  const int lane = threadIdx.x & 31, j = lane >> 2, q = lane & 3;
#pragma unroll
  for (int mt = 0; mt < C::TT; ++mt)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int slot = 16 * mt + 8 * r + j;
      const uint8_t* row = p.k.base + (size_t(__shfl_sync(0xffffffffu, at.k, slot)) << 4);
      if constexpr (C::KB == 16) {
#pragma unroll
        for (int c = 0; c < C::DP / 32; ++c) {
          if (32 * c + 8 * q < p.d) ldg_words<4>(&f.k[mt][r][4 * c], row + 64 * c + 16 * q);
          else f.k[mt][r][4 * c] = f.k[mt][r][4 * c + 1] = f.k[mt][r][4 * c + 2] = f.k[mt][r][4 * c + 3] = 0u;
        }
      } else {
        constexpr int n = C::KB == 8 ? 4 : 2;
#pragma unroll
        for (int g = 0; g < C::NG; ++g) ldg_words<n>(&f.k[mt][r][n * g], row + 4 * n * (4 * g + q));
      }
    }
  if constexpr (C::Q) load_scales<C::NG>(f.ks, f.kb, p.ks, at.ks, (at.valid >> (lane & (C::TS - 1))) & 1u);
}

template <class C>
__device__ __forceinline__ void load_v(const PagedView& p, const PagedPlace& at, PagedTile<C>& f) {
  const int lane = threadIdx.x & 31, j = lane >> 2, q = lane & 3;
#pragma unroll
  for (int mt = 0; mt < C::TT; ++mt) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // slots 2q, 2q + 1, 2q + 8, 2q + 9
      const int slot = 16 * mt + 2 * q + (e & 1) + 8 * (e >> 1);
      const uint8_t* row = p.v.base + (size_t(__shfl_sync(0xffffffffu, at.v, slot)) << 4);
      constexpr int n = C::VB == 16 ? 4 : C::VB == 8 ? 2 : 1;
#pragma unroll
      for (int g = 0; g < C::NG; ++g) {
        if (C::VB != 16 || 64 * g + 8 * j < p.d) {
          ldg_words<n>(&f.v[mt][e][n * g], row + 4 * n * (8 * g + j));
        } else {
#pragma unroll
          for (int i = 0; i < n; ++i) f.v[mt][e][n * g + i] = 0u;
        }
      }
    }
  }
  if constexpr (C::Q) load_scales<C::NG>(f.vs, f.vb, p.vs, at.vs, (at.valid >> (lane & (C::TS - 1))) & 1u);
}

// The segment's queries into shared memory; codes: scaled fp16, group sums.
template <class C>
__device__ __forceinline__ void load_queries(const PagedView& p, const PagedAttnArgs& a, const PagedSeg& s,
                                             PagedSmem<C>& sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int hb = s.hh - s.h * a.HB;
  for (int n = warp; n < C::HN; n += C::W) {
    const int g = hb * C::HN + n;
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    const bool in = g < a.G && 8 * lane < p.d;
    if (in) x = *reinterpret_cast<const uint4*>(a.q + s.b * a.q_b + int64_t(s.h * a.G + g) * a.q_h + 8 * lane);
    if constexpr (!C::Q) {
      if (8 * lane < C::DP) *reinterpret_cast<uint4*>(&sm.q[n][8 * lane]) = x;
    } else {
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      float y[8], top = 0.0f, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 u = unpack16<false>(w[i]);
        y[2 * i] = u.x;
        y[2 * i + 1] = u.y;
        top = fmaxf(top, fmaxf(fabsf(u.x), fabsf(u.y)));
      }
      top = bfly_max(top);
      const int e = min(247, max(7, int(__float_as_uint(top) >> 23)));  // 2^(e - 127) <= top < 2^(e - 126)
      const float f = __int_as_float((254 - e) << 23);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = __half2float(__float2half_rn(y[i] * f));
        sum += y[i];
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (8 * lane < C::DP) {
        // 4-bit codes come out as pairs (i, i + 4)
        constexpr bool four = C::KB == 4;
        *reinterpret_cast<uint4*>(&sm.q[n][8 * lane]) =
            four ? make_uint4(pack16<true>(y[0], y[4]), pack16<true>(y[1], y[5]), pack16<true>(y[2], y[6]),
                              pack16<true>(y[3], y[7]))
                 : make_uint4(pack16<true>(y[0], y[1]), pack16<true>(y[2], y[3]), pack16<true>(y[4], y[5]),
                              pack16<true>(y[6], y[7]));
        if ((lane & 7) == 0) sm.qsum[n][lane >> 3] = sum;
      }
      if (lane == 0) sm.qfac[n] = __int_as_float(e << 23);
    }
  }
}

// A warp's running state of HN heads: lane (j, q) holds heads 2q, 2q + 1 of
// each n tile; acc[nt][g][i][.] dims 64 g + 8 j + 2 i (+ 1) of both.
template <class C>
struct PagedState {
  float m[C::NT][2], mu[C::NT][2], l[C::NT][2];  // maximum, the reference in use (0 while m is -inf), lane's part of the sum
  float acc[C::NT][C::NG][4][4];
  float xb[C::NT][2][C::Q ? C::NG : 1];          // codes: sum of p * bias
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[nt][e] = -INFINITY;
        mu[nt][e] = l[nt][e] = 0.0f;
#pragma unroll
        for (int g = 0; g < (C::Q ? C::NG : 1); ++g) xb[nt][e][g] = 0.0f;
      }
#pragma unroll
      for (int g = 0; g < C::NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[nt][g][i][c] = 0.0f;
    }
  }
};

// S^T of a tile: x[mt][nt] in the layout of the MMA's result (rows j, j + 8;
// heads 2q, 2q + 1), in log2 units.
template <class C>
__device__ __forceinline__ void tile_scores(const PagedAttnArgs& a, const PagedSmem<C>& sm, const PagedTile<C>& f,
                                            float (&x)[C::TT][C::NT][4]) {
  const int lane = threadIdx.x & 31, j = lane >> 2, q = lane & 3;
#pragma unroll
  for (int mt = 0; mt < C::TT; ++mt)
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[mt][nt][i] = 0.0f;
  if constexpr (!C::Q) {
#pragma unroll
    for (int c = 0; c < C::DP / 32; ++c)
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt) {
        const uint4 b = *reinterpret_cast<const uint4*>(&sm.q[8 * nt + j][32 * c + 8 * q]);
#pragma unroll
        for (int mt = 0; mt < C::TT; ++mt) {
          const uint32_t* k0 = &f.k[mt][0][4 * c];
          const uint32_t* k1 = &f.k[mt][1][4 * c];
          mma16816<C::F16>(x[mt][nt], k0[0], k1[0], k0[1], k1[1], b.x, b.y);
          mma16816<C::F16>(x[mt][nt], k0[2], k1[2], k0[3], k1[3], b.z, b.w);
        }
      }
  } else {
    uint32_t ks[C::TT][2][C::SW], kb[C::TT][2][C::SW];
#pragma unroll
    for (int mt = 0; mt < C::TT; ++mt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        from_lane(ks[mt][r], f.ks, 16 * mt + 8 * r + j);
        from_lane(kb[mt][r], f.kb, 16 * mt + 8 * r + j);
      }
#pragma unroll
    for (int g = 0; g < C::NG; ++g) {
      float d[C::TT][C::NT][4];
#pragma unroll
      for (int mt = 0; mt < C::TT; ++mt)
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) d[mt][nt][i] = 0.0f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // 8 of the lane's 16 dims: two k steps
        uint32_t A[C::TT][2][4];              // per row: the pairs of k steps 0 and 1
#pragma unroll
        for (int mt = 0; mt < C::TT; ++mt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if constexpr (C::KB == 8) {
              const uint32_t w0 = f.k[mt][r][4 * g + 2 * half], w1 = f.k[mt][r][4 * g + 2 * half + 1];
              A[mt][r][0] = byte_pair<0x4140>(w0);
              A[mt][r][1] = byte_pair<0x4342>(w0);
              A[mt][r][2] = byte_pair<0x4140>(w1);
              A[mt][r][3] = byte_pair<0x4342>(w1);
            } else {
              const uint32_t w = f.k[mt][r][2 * g + half];
              A[mt][r][0] = nib_even(w);
              A[mt][r][1] = nib_odd(w);
              A[mt][r][2] = nib_even(w >> 8);
              A[mt][r][3] = nib_odd(w >> 8);
            }
          }
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
          const uint4 b = *reinterpret_cast<const uint4*>(&sm.q[8 * nt + j][64 * g + 16 * q + 8 * half]);
#pragma unroll
          for (int mt = 0; mt < C::TT; ++mt) {
            mma16816<true>(d[mt][nt], A[mt][0][0], A[mt][1][0], A[mt][0][1], A[mt][1][1], b.x, b.y);
            mma16816<true>(d[mt][nt], A[mt][0][2], A[mt][1][2], A[mt][0][3], A[mt][1][3], b.z, b.w);
          }
        }
      }
      constexpr float mid = C::KB == 8 ? 128.0f : 8.0f;
#pragma unroll
      for (int mt = 0; mt < C::TT; ++mt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float sc = scale_of(ks[mt][r], g), bi = __fmaf_rn(mid, sc, scale_of(kb[mt][r], g));
#pragma unroll
          for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float& y = x[mt][nt][2 * r + e];
              y = __fmaf_rn(sc, d[mt][nt][2 * r + e], __fmaf_rn(bi, sm.qsum[8 * nt + 2 * q + e][g], y));
            }
        }
    }
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float fac = sm.qfac[8 * nt + 2 * q + e];
#pragma unroll
        for (int mt = 0; mt < C::TT; ++mt) {
          x[mt][nt][e] *= fac;
          x[mt][nt][2 + e] *= fac;
        }
      }
  }
#pragma unroll
  for (int mt = 0; mt < C::TT; ++mt)
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[mt][nt][i] = a.cap_out != 0.0f ? a.cap_out * tanhf(x[mt][nt][i] * a.cap_in) : x[mt][nt][i] * a.scale_log2;
}

// The tile's slots into the state: x becomes p.
template <class C>
__device__ __forceinline__ void tile_fold(PagedTile<C>& f, uint32_t valid, float (&x)[C::TT][C::NT][4],
                                          PagedState<C>& st) {
  const int lane = threadIdx.x & 31, j = lane >> 2, q = lane & 3;
  constexpr uint32_t full = C::TS == 32 ? 0xffffffffu : (1u << C::TS) - 1u;
  if (valid != full) {
    // slots past the end: score -inf, and nothing of their rows' bits enters
#pragma unroll
    for (int mt = 0; mt < C::TT; ++mt) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (!((valid >> (16 * mt + 8 * r + j)) & 1u)) {
#pragma unroll
          for (int nt = 0; nt < C::NT; ++nt) x[mt][nt][2 * r] = x[mt][nt][2 * r + 1] = -INFINITY;
        }
      if constexpr (!C::Q) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!((valid >> (16 * mt + 2 * q + (e & 1) + 8 * (e >> 1))) & 1u)) {
#pragma unroll
            for (int i = 0; i < C::VW; ++i) f.v[mt][e][i] = 0u;
          }
      }
    }
  }
  // the reference follows the maximum when it is passed by more than LAG
  float es[C::TT][2];  // codes: log2 of the largest |scale| of rows j, j + 8, below by less than 1
  if constexpr (C::Q) {
    float big = 0.0f;
#pragma unroll
    for (int g = 0; g < C::NG; ++g) big = fmaxf(big, fabsf(scale_of(f.vs, g)));
    // (rec_kv_append's scales are 2^-24 or more; the bounds keep two references' distance inside ex2's range)
    const float own = float(min(96, max(-24, int(__float_as_uint(big) >> 23) - 127)));
#pragma unroll
    for (int mt = 0; mt < C::TT; ++mt)
#pragma unroll
      for (int r = 0; r < 2; ++r) es[mt][r] = __shfl_sync(0xffffffffu, own, 16 * mt + 8 * r + j);
  }
  float top[C::NT][2];
  bool move = false;
#pragma unroll
  for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float t = -INFINITY;
#pragma unroll
      for (int mt = 0; mt < C::TT; ++mt)
#pragma unroll
        for (int r = 0; r < 2; ++r) t = fmaxf(t, C::Q ? x[mt][nt][2 * r + e] + es[mt][r] : x[mt][nt][2 * r + e]);
      top[nt][e] = t;
      move |= t > st.m[nt][e] + C::LAG;
    }
  if (__any_sync(0xffffffffu, move)) {
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float t = top[nt][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
        const float mn = fmaxf(st.m[nt][e], t);
        // codes: whole, so that states are brought to another reference by powers of two
        const float mu = mn == -INFINITY ? 0.0f : (C::Q ? floorf(mn) : mn) - C::REF;
        const float al = st.m[nt][e] == -INFINITY ? 0.0f : ex2(st.mu[nt][e] - mu);  // (the state is 0 then)
        st.m[nt][e] = mn;
        st.mu[nt][e] = mu;
        st.l[nt][e] *= al;
        if constexpr (C::Q) {
#pragma unroll
          for (int g = 0; g < C::NG; ++g) st.xb[nt][e][g] *= al;
        }
#pragma unroll
        for (int g = 0; g < C::NG; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            st.acc[nt][g][i][e] *= al;
            st.acc[nt][g][i][2 + e] *= al;
          }
      }
  }
#pragma unroll
  for (int mt = 0; mt < C::TT; ++mt)
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[mt][nt][i] = ex2(x[mt][nt][i] - st.mu[nt][i & 1]);
        st.l[nt][i & 1] += x[mt][nt][i];
      }
  // O^T += V^T P^T
#pragma unroll
  for (int mt = 0; mt < C::TT; ++mt) {
    uint32_t hi[C::NT][2], lo[C::NT][2];
    auto split = [&](int nt, float w0, float w1, float w2, float w3) {
      const uint32_t h0 = pack16<C::F16>(w0, w1), h1 = pack16<C::F16>(w2, w3);
      hi[nt][0] = trans8x8(h0);
      hi[nt][1] = trans8x8(h1);
      const float2 u0 = unpack16<C::F16>(h0), u1 = unpack16<C::F16>(h1);
      lo[nt][0] = trans8x8(pack16<C::F16>(w0 - u0.x, w1 - u0.y));
      lo[nt][1] = trans8x8(pack16<C::F16>(w2 - u1.x, w3 - u1.y));
    };
    if constexpr (!C::Q) {
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt) split(nt, x[mt][nt][0], x[mt][nt][1], x[mt][nt][2], x[mt][nt][3]);
    }
    uint32_t vs[2][C::SW], vb[2][C::SW];
    if constexpr (C::Q) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        from_lane(vs[r], f.vs, 16 * mt + 8 * r + j);
        from_lane(vb[r], f.vb, 16 * mt + 8 * r + j);
      }
    }
#pragma unroll
    for (int g = 0; g < C::NG; ++g) {
      if constexpr (C::Q) {
        constexpr float mid = C::VB == 8 ? 128.0f : 8.0f;
        const float s0 = scale_of(vs[0], g), s1 = scale_of(vs[1], g);
        const float b0 = __fmaf_rn(mid, s0, scale_of(vb[0], g)), b1 = __fmaf_rn(mid, s1, scale_of(vb[1], g));
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
          const float* pp = x[mt][nt];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            st.xb[nt][e][g] = __fmaf_rn(pp[e], b0, __fmaf_rn(pp[2 + e], b1, st.xb[nt][e][g]));
          split(nt, pp[0] * s0, pp[1] * s0, pp[2] * s1, pp[3] * s1);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // dims 2i, 2i + 1 of the lane's 8
        uint32_t A[4];
        if constexpr (C::VB == 16) {
          const uint32_t v0 = f.v[mt][0][4 * g + i], v1 = f.v[mt][1][4 * g + i];
          const uint32_t v2 = f.v[mt][2][4 * g + i], v3 = f.v[mt][3][4 * g + i];
          A[0] = prmt(v0, v1, 0x5410);
          A[1] = prmt(v0, v1, 0x7632);
          A[2] = prmt(v2, v3, 0x5410);
          A[3] = prmt(v2, v3, 0x7632);
        } else if constexpr (C::VB == 8) {
          const int w = 2 * g + (i >> 1);
          const uint32_t sel = i & 1 ? 0x7362 : 0x5140;
          const uint32_t y0 = prmt(f.v[mt][0][w], f.v[mt][1][w], sel), y1 = prmt(f.v[mt][2][w], f.v[mt][3][w], sel);
          A[0] = byte_pair<0x4140>(y0);
          A[1] = byte_pair<0x4342>(y0);
          A[2] = byte_pair<0x4140>(y1);
          A[3] = byte_pair<0x4342>(y1);
        } else {
          const uint32_t sel = i < 2 ? 0x5410 : 0x7632;
          uint32_t y0 = prmt(f.v[mt][0][g], f.v[mt][1][g], sel), y1 = prmt(f.v[mt][2][g], f.v[mt][3][g], sel);
          if (i & 1) {
            y0 >>= 8;
            y1 >>= 8;
          }
          A[0] = nib_even(y0);
          A[1] = nib_odd(y0);
          A[2] = nib_even(y1);
          A[3] = nib_odd(y1);
        }
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
          mma16816<C::F16>(st.acc[nt][g][i], A[0], A[1], A[2], A[3], hi[nt][0], hi[nt][1]);
          mma16816<C::F16>(st.acc[nt][g][i], A[0], A[1], A[2], A[3], lo[nt][0], lo[nt][1]);
        }
      }
    }
  }
}

// Length of session b, clamped to the table (a longer one is reported).
__device__ __forceinline__ int session_length(const PagedView& p, const int* lengths, int b, int* status) {
  const int L = lengths[b];
  if (L >= 0 && L <= p.slots) return L;
  report(status, kStatusBadPage);
  return L < 0 ? 0 : int(p.slots);
}

// len[b] and pre[b], the units of the sessions before b (at least one each).
template <class F>
__device__ __forceinline__ void plan_units(const PagedView& p, const int* lengths, int* status, int threads, int* len,
                                           int* pre, int* scan, F units) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int carry = 0;
  for (int b0 = 0; b0 < p.batch; b0 += threads) {
    const int b = b0 + int(threadIdx.x);
    int n = 0;
    if (b < p.batch) {
      len[b] = session_length(p, lengths, b, status);
      n = units(len[b]);
    }
    int y = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    if (lane == 31) scan[warp] = y;
    __syncthreads();
    int before = carry, all = carry;
    for (int w = 0; w < threads / 32; ++w) {
      if (w < warp) before += scan[w];
      all += scan[w];
    }
    if (b < p.batch) pre[b] = before + y - n;
    carry = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) pre[p.batch] = carry;
  __syncthreads();
}
// The session whose units hold index u of a list with H copies of each.
__device__ __forceinline__ int unit_session(const int* pre, int batch, int64_t H, int64_t u) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] * H <= u) lo = mid; else hi = mid;
  }
  return lo;
}

template <class C>
__global__ void __launch_bounds__(C::W * 32, C::MINB) k_paged_attn(const PagedView p, const PagedAttnArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  PagedSmem<C>& sm = *reinterpret_cast<PagedSmem<C>*>(smem_raw);
  int* len = reinterpret_cast<int*>(smem_raw + sizeof(PagedSmem<C>));
  int* pre = len + p.batch;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = lane >> 2, q = lane & 3;
  auto first_slot = [&](int L) { return a.window > 0 ? max(0, L - a.window) : 0; };
  plan_units(p, a.lengths, blockIdx.x == 0 ? a.status : nullptr, C::W * 32, len, pre, sm.scan,
             [&](int L) { return max(1, (L - first_slot(L) + C::UT - 1) / C::UT); });
  const int64_t H = int64_t(p.hkv) * a.HB;
  {
    int64_t per = (pre[p.batch] * H + gridDim.x - 1) / gridDim.x;
    if (int64_t(p.batch) * H <= gridDim.x) {
      const int b = threadIdx.x, nb = b < p.batch ? pre[b + 1] - pre[b] : 0, most = int(per) + C::WHOLE;
      for (int k = int(per); k <= most; ++k)
        if (!__syncthreads_or(nb > k)) {  // every head's units filled up to k: a block's share is a head
          if (b <= p.batch) pre[b] = b * k;
          per = k;
          break;
        }
    }
    if (threadIdx.x == 0) sm.per = per;  // (held there: the loop below has no registers to spare)
    __syncthreads();
  }
  const int64_t total = pre[p.batch] * H;
  int64_t u = int64_t(blockIdx.x) * sm.per;
  auto end = [&] { return min(total, int64_t(blockIdx.x + 1) * sm.per); };
  if (u >= end()) return;

  auto seg_at = [&](int b, int hh, int ul, int64_t at) {
    PagedSeg s;
    s.b = b;
    s.hh = hh;
    s.h = hh / a.HB;
    s.L = len[b];
    s.lo = first_slot(s.L);
    s.nb = pre[b + 1] - pre[b];
    s.ul = ul;
    s.n = int(min(int64_t(s.nb - ul), end() - at));
    return s;
  };
  PagedSeg s;
  {
    const int b = unit_session(pre, p.batch, H, u);
    const int64_t rest = u - pre[b] * H;
    const int nb = pre[b + 1] - pre[b];
    s = seg_at(b, int(rest / nb), int(rest % nb), u);
  }
  auto tile_start = [&](const PagedSeg& g, int i) { return g.lo + ((g.ul + i) * C::W + warp) * C::TS; };

  PagedTile<C> f;
  PagedPlace at;
  find_places<C>(p, a, s, tile_start(s, 0), at);
  uint32_t valid = at.valid;
  if (valid) {
    load_k<C>(p, at, f);
    load_v<C>(p, at, f);
  }
  while (true) {
    PagedSeg ns = s;
    const bool more = u + s.n < end();
    if (more) {
      const bool wrap = s.hh + 1 == H;  // a block's units of one head are one segment
      ns = seg_at(wrap ? s.b + 1 : s.b, wrap ? 0 : s.hh + 1, 0, u + s.n);
    }
    load_queries<C>(p, a, s, sm);
    __syncthreads();
    PagedState<C> st;
    st.clear();
    for (int i = 0; i < s.n; ++i) {
      const int t0 = tile_start(s, i);
      at.valid = 0u;
      if (i + 1 < s.n) find_places<C>(p, a, s, tile_start(s, i + 1), at);
      else if (more) find_places<C>(p, a, ns, tile_start(ns, 0), at);
      if constexpr (!C::Q) {
        if (sm.per > 16) {
          if (i + 2 < s.n) prefetch_tile<C>(p, s, tile_start(s, i + 2));
          else if (more && i + 2 - s.n < ns.n) prefetch_tile<C>(p, ns, tile_start(ns, i + 2 - s.n));
        }
      }
      float x[C::TT][C::NT][4];
      if (valid) tile_scores<C>(a, sm, f, x);
      if (at.valid) load_k<C>(p, at, f);
      if (valid) {
        if (a.scores) {
          const int g0 = (s.hh - s.h * a.HB) * C::HN;
          float* sc = a.scores + (int64_t(s.b * p.hkv + s.h) * a.score_len + t0) * a.G + g0;
#pragma unroll
          for (int mt = 0; mt < C::TT; ++mt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int slot = 16 * mt + 8 * (c >> 1) + j;
#pragma unroll
              for (int nt = 0; nt < C::NT; ++nt) {
                const int g = 8 * nt + 2 * q + (c & 1);
                if (((valid >> slot) & 1u) && g0 + g < a.G) sc[int64_t(slot) * a.G + g] = x[mt][nt][c];
              }
            }
        }
        tile_fold<C>(f, valid, x, st);
      }
      if (at.valid) load_v<C>(p, at, f);
      valid = at.valid;
    }
    // ---- the warps' states meet in shared memory
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int n = 8 * nt + 2 * q + e;
        float l = st.l[nt][e];
        float xb[C::Q ? C::NG : 1];
#pragma unroll
        for (int g = 0; g < (C::Q ? C::NG : 1); ++g) xb[g] = st.xb[nt][e][g];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          l += __shfl_xor_sync(0xffffffffu, l, o);
          if constexpr (C::Q) {
#pragma unroll
            for (int g = 0; g < C::NG; ++g) xb[g] += __shfl_xor_sync(0xffffffffu, xb[g], o);
          }
        }
        float M = st.m[nt][e] == -INFINITY ? -INFINITY : st.mu[nt][e], back = 1.0f;
        if constexpr (C::Q) {
          if (l != 0.0f) {  // from the slots' scales' units to a sum in [1, 2)
            const int ex = min(126, max(-126, int(__float_as_uint(l) >> 23 & 255u) - 127));
            M += float(ex);
            back = __int_as_float((127 - ex) << 23);
          }
        }
        if (j == 0) {
          sm.m[warp][n] = M;
          sm.l[warp][n] = l * back;
        }
#pragma unroll
        for (int g = 0; g < C::NG; ++g) {
          float y[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[2 * i] = st.acc[nt][g][i][e];
            y[2 * i + 1] = st.acc[nt][g][i][2 + e];
          }
          if constexpr (C::Q) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = (y[i] + xb[g]) * back;
          }
          float4* dst = reinterpret_cast<float4*>(&sm.acc[warp][n][64 * g + 8 * j]);
          dst[0] = make_float4(y[0], y[1], y[2], y[3]);
          dst[1] = make_float4(y[4], y[5], y[6], y[7]);
        }
      }
    __syncthreads();
    const int g0 = (s.hh - s.h * a.HB) * C::HN;
    const int heads = min(C::HN, a.G - g0);
    const bool whole = s.n == s.nb;
    const int64_t head0 = pre[s.b] * H + int64_t(s.hh) * s.nb;  // first unit of this head
    // one thread per 4 dims of a head; (M, l, o) of the block
    auto write = [&](int n, int d, float M, float l, float4 o) {
      const int hq = s.h * a.G + g0 + n;
      const float sink = a.sinks ? bf(a.sinks[hq]) * kLog2e : -INFINITY;
      const float top = fmaxf(M, sink), ref = top == -INFINITY ? 0.0f : top;
      const float w = ex2(M - ref), sum = __fmaf_rn(l, w, ex2(sink - ref));
      const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(w, sum);
      if (d < p.d) {
        uint2 y;
        if (p.fp16) y = make_uint2(pack16<true>(o.x * inv, o.y * inv), pack16<true>(o.z * inv, o.w * inv));
        else y = make_uint2(pack16<false>(o.x * inv, o.y * inv), pack16<false>(o.z * inv, o.w * inv));
        *reinterpret_cast<uint2*>(a.out + s.b * a.o_b + hq * a.o_h + d) = y;
      }
      if (d == 0 && (a.lse || a.lse2)) {
        const float lse2 = sum == 0.0f ? -INFINITY : ref + log2f(sum);
        if (a.lse) a.lse[s.b * a.hq + hq] = lse2 * kLn2;
        // (every score -inf: 2^(-inf - 0) gives the slots no weight)
        if (a.lse2) a.lse2[s.b * a.hq + hq] = sum == 0.0f ? 0.0f : lse2;
      }
    };
    const int slot = whole ? 0 : 2 * blockIdx.x + (int64_t(blockIdx.x) * sm.per >= head0 ? 0 : 1);
    for (int i = threadIdx.x; i < heads * (C::DP / 4); i += C::W * 32) {
      const int n = i / (C::DP / 4), d = 4 * (i % (C::DP / 4));
      float M = sm.m[0][n];
#pragma unroll
      for (int w = 1; w < C::W; ++w) M = fmaxf(M, sm.m[w][n]);
      const float ref = M == -INFINITY ? 0.0f : M;
      float l = 0.0f;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < C::W; ++w) {
        const float al = ex2(sm.m[w][n] - ref);
        const float4 y = *reinterpret_cast<const float4*>(&sm.acc[w][n][d]);
        l = __fmaf_rn(sm.l[w][n], al, l);
        o.x = __fmaf_rn(y.x, al, o.x);
        o.y = __fmaf_rn(y.y, al, o.y);
        o.z = __fmaf_rn(y.z, al, o.z);
        o.w = __fmaf_rn(y.w, al, o.w);
      }
      if (whole) {
        write(n, d, M, l, o);
      } else {
        __stcg(reinterpret_cast<float4*>(a.part_acc + (int64_t(slot) * C::HN + n) * C::DP + d), o);
        if (d == 0) __stcg(a.part_ml + int64_t(slot) * C::HN + n, make_float2(M, l));
      }
    }
    if (!whole) {
      // the last of the head's blocks joins their partials, in block order
      __syncthreads();
      const int c0 = int(head0 / sm.per), c1 = int((head0 + s.nb - 1) / sm.per), parts = c1 - c0 + 1;
      if (threadIdx.x == 0) {
        unsigned* c = a.counters + s.b * H + s.hh;
        // releases the block's partials (the barrier above orders them before), acquires the others'
        unsigned before;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(c) : "memory");
        sm.last = before == unsigned(parts - 1);
        if (sm.last) *c = 0u;
      }
      __syncthreads();
      if (sm.last) {
        float* wgt = &sm.acc[0][0][0];  // [HN][parts]
        auto part_slot = [&](int c) { return 2 * c + (int64_t(c) * sm.per >= head0 ? 0 : 1); };
        for (int n = warp; n < heads; n += C::W) {
          float M = -INFINITY;
          for (int c = lane; c < parts; c += 32) M = fmaxf(M, __ldcg(a.part_ml + int64_t(part_slot(c0 + c)) * C::HN + n).x);
          M = bfly_max(M);
          const float ref = M == -INFINITY ? 0.0f : M;
          float l = 0.0f;
          for (int c = lane; c < parts; c += 32) {
            const float2 ml = __ldcg(a.part_ml + int64_t(part_slot(c0 + c)) * C::HN + n);
            const float w = ex2(ml.x - ref);
            wgt[n * parts + c] = w;
            l = __fmaf_rn(ml.y, w, l);
          }
          l = bfly_sum(l);
          if (lane == 0) {
            sm.head_m[n] = M;
            sm.head_l[n] = l;
          }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < heads * (C::DP / 4); i += C::W * 32) {
          const int n = i / (C::DP / 4), d = 4 * (i % (C::DP / 4));
          float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
          for (int c = 0; c < parts; ++c) {
            const float4 y = __ldcg(reinterpret_cast<const float4*>(
                a.part_acc + (int64_t(part_slot(c0 + c)) * C::HN + n) * C::DP + d));
            const float w = wgt[n * parts + c];
            o.x = __fmaf_rn(y.x, w, o.x);
            o.y = __fmaf_rn(y.y, w, o.y);
            o.z = __fmaf_rn(y.z, w, o.z);
            o.w = __fmaf_rn(y.w, w, o.w);
          }
          write(n, d, sm.head_m[n], sm.head_l[n], o);
        }
      }
    }
    u += s.n;
    if (!more) break;
    s = ns;
    __syncthreads();  // shared memory is reused by the next segment
  }
}

// Launches the configuration's kernel over `sms` SMs.
template <class C>
cudaError_t launch_paged_attn(const PagedView& p, const PagedAttnArgs& a, int sms, cudaStream_t st) {
  const size_t smem = sizeof(PagedSmem<C>) + size_t(2 * p.batch + 1) * sizeof(int);
  // the limit covers the largest batch, so it is set once
  const cudaError_t e = set_smem_limit(reinterpret_cast<const void*>(&k_paged_attn<C>),
                                       sizeof(PagedSmem<C>) + size_t(2 * kPagedMaxBatch + 1) * sizeof(int));
  if (e != cudaSuccess) return e;
  k_paged_attn<C><<<sms * C::MINB, C::W * 32, smem, st>>>(p, a);
  return cudaGetLastError();
}

// Which configuration a cache takes; defined in paged_attn_*.cu.
struct PagedAttnShape {
  int dp, hn, blocks;  // padded head dim, heads of a block, blocks per SM
};
PagedAttnShape paged_attn_shape(const PagedView& p, int group);
cudaError_t paged_attn_bf16(const PagedView& p, const PagedAttnArgs& a, int sms, cudaStream_t st);
cudaError_t paged_attn_fp16(const PagedView& p, const PagedAttnArgs& a, int sms, cudaStream_t st);
cudaError_t paged_attn_codes8(const PagedView& p, const PagedAttnArgs& a, int sms, cudaStream_t st);  // K 8 bit
cudaError_t paged_attn_codes4(const PagedView& p, const PagedAttnArgs& a, int sms, cudaStream_t st);  // K 4 bit

// DP and NT of a shape: 8 or 16 heads a block; 8 at the widest rows, whose
// state of 16 would not fit the registers.
template <template <int, int> class Cfg>
cudaError_t paged_attn_by_shape(const PagedView& p, const PagedAttnArgs& a, int sms, cudaStream_t st) {
  const PagedAttnShape s = paged_attn_shape(p, a.G);
  if (s.dp == 64)
    return s.hn == 8 ? launch_paged_attn<typename Cfg<64, 1>::type>(p, a, sms, st)
                     : launch_paged_attn<typename Cfg<64, 2>::type>(p, a, sms, st);
  if (s.dp == 128)
    return s.hn == 8 ? launch_paged_attn<typename Cfg<128, 1>::type>(p, a, sms, st)
                     : launch_paged_attn<typename Cfg<128, 2>::type>(p, a, sms, st);
  return launch_paged_attn<typename Cfg<256, 1>::type>(p, a, sms, st);
}
// Warps of a block by the registers a thread needs (65,536 of an SM).
constexpr int paged_warps(int dp, int nt) { return dp * nt <= 128 ? 12 : 8; }

}  // namespace rec
