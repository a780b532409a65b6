// tree_decode.cuh -- the split kernel of tree_decode (include/wfattn.h), one
// instantiation a row format, head size, query type and number of query rows.
//
// The rows of queries that share one cache head, R = heads_q / heads * nodes,
// are attended together, up to 32 in a tile: every cache row is read once a tile.
// The kernel works on transposed products, whose narrow side (8) holds queries:
//
//   S^T [16 keys x 8 queries] = K [16 x D] Q^T [D x 8]
//   O^T [D x 8 queries]      += V^T [D x 16 keys] P^T [16 x 8]
//
// with mma.sync: rows of K and V go from shared memory through a conversion in
// registers (codes to f16; nothing is written back), which tcgen05 operands in
// shared or tensor memory would need a round trip for, and there are up to 32
// query rows where a tcgen05 tile has 128 (more: tree_decode_wide.cuh).  Products:
//  * e4m3 / int4 rows: the codes (int4: u - 8) are exact in f16; scale and
//    minimum of a row are applied to the f32 score and to the f32 weight;
//  * bf16 rows: bf16 products, the weights as two bf16 terms (16 bits);
//  * f32 rows: tf32 products of two-term splits (hi hi, hi lo, lo hi), and
//    with f32 queries over quantised rows Q and P as two f16 terms: ~2^-21.
// Queries are scaled by a power of two into f16's upper range, weights are
// taken as p <= 2^4 times the row's scale over the running largest one that the
// query sees, also in f16's range; sums, maxima and all other arithmetic are f32.
//
// Softmax is online with a lazy maximum: weights are 2^(s - m) for a reference
// m that is raised (and the sums rescaled) only when a score passes m + 4, so
// most tiles pay one vote instead of the maximum's shuffles.
//
// Work: a unit is kKeys keys of one (sequence, cache head, tile of query
// rows); the units of all sequences in order are dealt in equal contiguous
// shares to a grid of kCtas CTAs an SM, whatever the lengths (short segments
// whole).  A CTA streams its units through a ring of cp.async stages without
// regard to where a segment (one sequence, head and tile) ends; a segment that
// lies in one CTA is written out directly.  Of the others every CTA writes its part (maximum,
// sum, unnormalised output) to the workspace, and they are joined in their order:
// the same bits every time.  With one or two rows the CTA whose part is the last
// to arrive, by a counter, does that, without another launch; more rows would
// keep that CTA busy (8 rows of 128 values in 27 parts 15 us, 60 rows in 7 parts
// 40 us), so there a second kernel does.
// Four warps split the keys of a unit or, with more rows, the rows.
//
// HBM bounds it where the conversion is short; where it is not, the latency of
// unpacking, product, exponential and product with the 12 to 16 warps an SM that
// the registers leave (half the issue slots stay empty).  One token, ragged lengths:
// rows of 64 values, 64 x 25 heads, 145,700 keys of each, bf16 6.4 TB/s (145 us),
// e4m3 4.6 (107); rows of 128, 8 heads, 326,100 keys of each, e4m3 5.8 (119), 4 bits
// under 8 query heads 3.9 (90).
#pragma once

#include <float.h>
#include <math.h>

#include "cache_format.cuh"

namespace wfattn {
namespace tree {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kMaxSms = 148;  // CTAs are dealt for at most this many SMs

// Counters of arrived parts, at the start of the workspace: zero before the
// first launch on it, and left at zero by each (atomicInc wraps).
constexpr int kCounters = WFATTN_TREE_DECODE_ZEROED / sizeof(unsigned int);  // one a CTA

// The segment that begins in a CTA and goes on in others.
struct Split {
  int64_t all;  // units in all
  int b, h, tile, last;  // the segment (b < 0: none), its last CTA
};

struct Params {
  CacheView c;
  int RT;        // row tiles a head
  int R, G, T;   // query rows a head = G heads x T nodes
  uint32_t over_T;  // ceil(2^32 / T)
  bool q_vec, o_vec;  // rows of q (o) are aligned for vector loads (stores)
  bool apart;         // parts are joined by a second kernel
  int ctas;      // of the grid
  const uint8_t *q;
  uint8_t *o;
  Strides3 qs, os;
  const int32_t *lens, *counts;
  const uint64_t *tree;
  int64_t tree_stride;
  float scale_log2;
  unsigned int *arrived;  // [kCounters]
  Split *split;  // [ctas] (tree_decode_wide.cuh)
  float *part;   // [ctas][2][rows][D], then [ctas][2][rows][2] (maximum, sum)
  unsigned int *status;
};

// r / T, exact for r < 2^26: r (over_T T - 2^32) < r T stays below 2^32.
__device__ __forceinline__ int over_T(const Params &p, int r) {
  return p.T == 1 ? r : (int)__umulhi((uint32_t)r, p.over_T);
}

enum Kind { kF16, kBf16, kTf32 };

template <int kFmt_, int D_, bool kF32_, int kNT_, int kRW_>
struct Cfg {
  static constexpr int kFmt = kFmt_, D = D_, kNT = kNT_, kRW = kRW_, kKW = kWarps / kRW_;
  static constexpr bool kF32 = kF32_;  // queries and output
  static constexpr bool kWide = false;
  static constexpr Kind kKind = kFmt == WFATTN_CACHE_F32    ? kTf32
                                : kFmt == WFATTN_CACHE_BF16 ? kBf16
                                                            : kF16;
  static constexpr bool kScaled = CacheRow<kFmt, D>::kScaled;
  static constexpr int kRowBytes = CacheRow<kFmt, D>::kBytes;
  static constexpr int kRows = 8 * kNT * kRW;  // query rows of a CTA
  // keys of a unit: about 16 to 32 KB of K and V
  static constexpr int kKeys = kRowBytes == 32    ? 256
                               : kRowBytes == 64  ? (kNT * D > 128 ? 256 : 128)
                               : kRowBytes == 128 && (D == 64 || kNT == 2) ? 128
                                                                           : 64;
  // 16-key tiles taken together: two independent chains of products hide their
  // latency.  Rows of 128 values have two chains each, and smaller units leave
  // more of the stages in flight (e4m3, one token, 342k keys of 8 heads: 128 us
  // against 160 with two tiles and 128 keys).
  static constexpr int kKT = kRowBytes <= 64 || (kRowBytes == 128 && (D == 64 || kNT == 2)) ? 2 : 1;
  static constexpr int kGroups = kKeys / (16 * kKT * kKW);  // of a warp in a unit
  static constexpr int kKBytes = kKeys * kRowBytes;
  static constexpr int kMerge = kWarps * 8 * kNT * D * 4;  // sums of O, in a used stage
  static constexpr int kData = 2 * kKBytes + (kScaled ? 8 * kKeys : 0);
  static constexpr int kStage = kData > kMerge ? kData : kMerge;
  static constexpr int kStats = kWarps * 8 * kNT * 2 * 4;
  // CTAs an SM: as many as the registers of the fragments and two stages allow
  static constexpr int kCtas = kRowBytes >= 512                                     ? 1
                               : kRowBytes == 256 || (kF32 ? 2 : kNT) * D == 256 ? 2
                               : kNT * D <= 64 && kRowBytes <= 64                  ? 4
                                                                                    : 3;
  static constexpr int kFit = (227 * 1024 / kCtas - 2048 - kStats) / kStage;
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static_assert(kStages >= 2, "shared memory budget");
  static constexpr int kSmem = kStages * kStage + kStats;
  static constexpr int kMt = D / 16;  // row tiles of O^T
};

// ------------------------------------------------------------- instructions

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(live ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(live ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
template <bool kTrans>
__device__ __forceinline__ void ldmatrix4(uint32_t a, uint32_t (&r)[4]) {
  if constexpr (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
}
// The 8x8 matrix of 16-bit elements held by the warp, transposed.
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
template <Kind kKind>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  if constexpr (kKind == kF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else if constexpr (kKind == kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// (x & kMask) | kBits in one operation
template <uint32_t kMask, uint32_t kBits>
__device__ __forceinline__ uint32_t and_or(uint32_t x) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "n"(kMask), "n"(kBits));
  return r;
}
// 4-bit codes number 0 and 4 (kOdd: 1 and 5) of w as the f16x2 u - 8: a code
// put below f16's 1024 (above 64's sixteenths) reads 1024 + u (64 + u), exactly.
template <bool kOdd>
__device__ __forceinline__ uint32_t int4_f16x2(uint32_t w) {
  return kOdd ? hsub2(and_or<0x00f000f0u, 0x54005400u>(w), 0x54805480u)
              : hsub2(and_or<0x000f000fu, 0x64006400u>(w), 0x64086408u);
}
// f32 as tf32 terms: x to the nearest of 10 fraction bits (so that what the
// products cut from the rest has no sign of its own), and what is left (exact;
// the product unit takes its upper bits)
__device__ __forceinline__ uint32_t tf32_hi(uint32_t x) { return (x + 0x1000u) & 0xffffe000u; }
__device__ __forceinline__ uint32_t tf32_lo(uint32_t x) {
  return __float_as_uint(__uint_as_float(x) - __uint_as_float(tf32_hi(x)));
}

// ----------------------------------------------------------------- layouts

// Byte offset `o` of row `r` in a stage's K or V: 16-byte pieces are permuted
// inside 128-byte lines so that the loads of a fragment (8 rows, or 4 row
// pairs, at one offset) fall into different banks.
template <class C>
__host__ __device__ constexpr uint32_t swizzle_bits(uint32_t r) {  // linear in the bits of r
  return (C::kKind == kBf16     ? r & 7
          : C::kRowBytes >= 128 ? (r & 6) ^ ((r & 1) << 2)
          : C::kRowBytes == 64  ? r & 6
                                : (r >> 1) & 2)
         << 4;
}
template <class C>
__device__ __forceinline__ uint32_t swizzle(uint32_t r, uint32_t o) {
  return (r * C::kRowBytes + o) ^ swizzle_bits<C>(r);
}

// Which value the row g (r = 0) or g + 8 (r = 1) of O^T's tile mt is.
template <class C>
__device__ __forceinline__ int o_index(int mt, int g, int r) {
  if constexpr (C::kKind == kBf16) return 16 * mt + g + 8 * r;
  if constexpr (C::kKind == kTf32) return 4 * (g + 8 * (mt >> 1)) + 2 * (mt & 1) + r;
  return (C::D / 8) * g + 2 * mt + r;
}

// Place of value d of row r of the sums where warps meet: groups of four values
// are permuted so that a fragment's lanes write to different banks (two to one
// at most) and a row is still read four values at a time.
template <class C>
__device__ __forceinline__ int sum_index(int r, int d) {
  const int x = C::kKind == kBf16 ? r & 6 : C::kKind == kTf32 ? (r & 2) << 1 : r >> 1 & 3;
  return r * C::D + (d ^ (x << 2));
}

// One value of a V row in a stage, unscaled (used where a row is not finite).
template <class C>
__device__ __forceinline__ float v_value(uint32_t v, int row, int d) {
  if constexpr (C::kFmt == WFATTN_CACHE_F32) {
    return __uint_as_float(lds32(v + swizzle<C>(row, 4 * d)));
  } else if constexpr (C::kFmt == WFATTN_CACHE_BF16) {
    const uint32_t w = lds32(v + swizzle<C>(row, 2 * (d & ~1)));
    return d & 1 ? ptx::bf16_hi(w) : ptx::bf16_lo(w);
  } else {
    const uint32_t w = lds32(v + swizzle<C>(row, d & ~3)) >> (8 * (d & 3));
    return ptx::f16x2_to_f32(ptx::e4m3x2_to_f16x2(w & 0xff)).x;
  }
}

// -------------------------------------------------------------- work order

struct Seq {
  int len, total;  // rows before the tree, rows in all
  int n;           // nodes
  int units;       // of one segment, at least 1
};

template <int kKeys>
__device__ __forceinline__ Seq sequence(const Params &p, int b, bool report) {
  Seq s;
  const int L = (int)p.c.L;
  int len = p.lens[b], n = p.counts ? p.counts[b] : p.T;
  bool bad = len < 0 || n < 0 || n > p.T;
  len = max(len, 0);
  n = min(max(n, 0), p.T);
  bad = bad || len > L || n > L - len;
  len = min(len, L);
  n = min(n, L - len);
  if (bad && report) atomicOr(p.status, kDevBadRowMask);
  s.len = len;
  s.n = n;
  s.total = len + n;
  s.units = max(1, (s.total - 1) / kKeys + 1);
  return s;
}

// A position in the order of units: sequence, cache head, tile of query rows,
// unit of keys.
template <int kKeys>
struct Cursor {
  int b, h, tile, u;
  Seq s;
  // whether the next unit is another segment's
  __device__ __forceinline__ bool next(const Params &p) {
    if (++u < s.units) return false;
    u = 0;
    if (++tile < p.RT) return true;
    tile = 0;
    if (++h < (int)p.c.H) return true;
    h = 0;
    if (++b < (int)p.c.B) s = sequence<kKeys>(p, b, false);
    return true;
  }
};

// What the joining kernel needs to know of the segment at c, which begins with
// unit s0 and goes on to the CTA of its last unit: unit s lies in the last CTA x
// with total x / ctas <= s.
template <int kKeys>
__device__ __forceinline__ Split split_of(const Params &p, const Cursor<kKeys> &c, int64_t s0,
                                          int64_t all) {
  Split s;
  s.all = all;
  s.b = c.b;
  s.h = c.h;
  s.tile = c.tile;
  s.last = (int)(((s0 + c.s.units) * p.ctas - 1) / all);
  return s;
}

// total * x / parts, x <= parts <= kCounters; 64-bit divisions are long.
__device__ __forceinline__ int64_t part_of(int64_t total, int x, int parts) {
  if (total < (int64_t(1) << 32) / kCounters) return (uint32_t)total * (uint32_t)x / (uint32_t)parts;
  return total * x / parts;
}

constexpr int kShort = 4;

// Finds this CTA's share [begin, end) of the units and where it begins.  Where
// no segment has more than kShort units the shares are whole segments: a few
// units' difference in load costs less than joining parts.  All the block's warps
// call it; the sequences are shared out over its first kThreads threads.
template <int kKeys>
__device__ __forceinline__ Cursor<kKeys> share(const Params &p, int64_t &begin, int64_t &end,
                                               int64_t &all) {
  __shared__ int64_t warp_sum[kWarps], offset, stop;
  __shared__ Cursor<kKeys> found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int B = (int)p.c.B, per = (B + kThreads - 1) / kThreads;
  const int b0 = (int)imin64(B, (int64_t)threadIdx.x * per), b1 = min(B - b0, per) + b0;
  const int64_t HR = p.c.H * p.RT;
  int64_t mine = 0;
  int longest = 0;
  Seq s;
  for (int b = b0; b < b1; ++b) {
    s = sequence<kKeys>(p, b, blockIdx.x == 0);
    mine += s.units * HR;
    longest = max(longest, s.units);
  }
  int64_t upto = mine;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, upto, x);
    if (lane >= x) upto += y;
  }
  if (lane == 31 && warp < kWarps) warp_sum[warp] = upto;
  const bool whole = !__syncthreads_or(longest > kShort);
  all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += warp_sum[w];
    all += warp_sum[w];
  }
  // unit (or, with whole segments, segment) where the share begins and ends
  const int64_t total = whole ? B * HR : all;
  const int64_t from = part_of(total, blockIdx.x, p.ctas);
  const int64_t to = part_of(total, blockIdx.x + 1, p.ctas);
  int64_t at = upto - mine;  // first unit of this thread's sequences
  for (int b = b0; b < b1; ++b) {
    if (per > 1) s = sequence<kKeys>(p, b, false);
    const int64_t n = s.units * HR;
    const int64_t lo = whole ? b * HR : at, hi = whole ? lo + HR : at + n;
    if (from >= lo && from < hi) {
      const int64_t into = whole ? (from - lo) * s.units : from - lo;
      const int hr = into < (int64_t(1) << 32) ? (int)((uint32_t)into / (uint32_t)s.units)
                                               : (int)(into / s.units);
      offset = at + into;
      found.b = b;
      found.u = (int)(into - (int64_t)hr * s.units);
      found.h = hr / p.RT;
      found.tile = hr - found.h * p.RT;
      found.s = s;
    }
    if (to > lo && to <= hi) stop = whole ? at + (to - lo) * s.units : to;
    at += n;
  }
  __syncthreads();
  begin = offset;
  end = to > from ? stop : begin;
  return found;
}

// ------------------------------------------------------------------ kernel

// What a warp holds of a segment: 8 kNT query rows.  Lane 4 g + t has row g of a
// fragment's 8 (16: g and g + 8) and columns 2t, 2t + 1.
template <class C>
struct Warp {
  // product steps along a row are 16 values (4 a lane) or, in tf32, 8 (2)
  static constexpr int kSteps = C::kKind == kTf32 ? C::D / 8 : C::D / 16;
  static constexpr int kE = C::kKind == kTf32 ? 2 : 4;
  static constexpr int kQTerms = C::kKind == kF16 && C::kF32 ? 2 : 1;
  static constexpr int kPTerms = C::kKind == kBf16 || (C::kKind == kF16 && C::kF32) ? 2 : 1;
  uint32_t q[C::kNT][kSteps][2 * kQTerms];
  float o[C::kNT][C::kMt][4];
  // of queries 2t, 2t + 1 of each 8:
  float qf[C::kNT][2], qsum[C::kNT][2];  // score = product * qf; sum of q (int4)
  uint64_t word[C::kNT][2];
  float m[C::kNT][2], l[C::kNT][2], om[C::kNT][2];
  // f16 weights carry scale * vinv.  Among a tree's nodes it is each query's own, so
  // that a scale that it does not see leaves its weights their bits; only tails
  // need those, so they lie in shared memory, as what to add to the bits of vinv.
  float vinv;
  int *own;  // of the warp's 8 kNT queries

  __device__ __forceinline__ float own_vinv(int nt, int i) const {
    return __int_as_float(__float_as_int(vinv) + own[8 * nt + 2 * (threadIdx.x & 3) + i]);
  }

  // The values of one query row that this lane multiplies, step by step.  Any
  // order along a row will do as long as K's fragments have the same.
  __device__ __forceinline__ void load_row(const Params &p, int64_t at, float (&x)[kSteps][kE]) {
    const int t = threadIdx.x & 3;
    const float *qf32 = reinterpret_cast<const float *>(p.q) + at;
    const uint16_t *q16 = reinterpret_cast<const uint16_t *>(p.q) + at;
    if constexpr (C::kKind == kBf16) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint16_t *from = q16 + 16 * s + 8 * i + 2 * t;
          const uint32_t w = p.q_vec ? *reinterpret_cast<const uint32_t *>(from)
                                     : from[0] | (uint32_t)from[1] << 16;
          x[s][2 * i] = ptx::bf16_lo(w), x[s][2 * i + 1] = ptx::bf16_hi(w);
        }
      return;
    }
    // runs of consecutive values: 4 (tf32), 16 (e4m3), D/4 (int4)
    constexpr int kRun = C::kKind == kTf32 ? 4 : C::kFmt == WFATTN_CACHE_E4M3 ? 16 : C::D / 4;
#pragma unroll
    for (int j = 0; j < C::D / 4 / kRun; ++j) {
      const int from = kRun * (t + 4 * j);
      float y[kRun];
      if constexpr (C::kF32) {
        if (p.q_vec) {
#pragma unroll
          for (int i = 0; i < kRun; i += 4) {
            const float4 v = *reinterpret_cast<const float4 *>(qf32 + from + i);
            y[i] = v.x, y[i + 1] = v.y, y[i + 2] = v.z, y[i + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < kRun; ++i) y[i] = qf32[from + i];
        }
      } else {
        if (p.q_vec) {
#pragma unroll
          for (int i = 0; i < kRun; i += 8) {
            float v[8];
            const uint4 w = *reinterpret_cast<const uint4 *>(q16 + from + i);
            cache_values8<WFATTN_CACHE_BF16>(&w.x, 0, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i + e] = v[e];
          }
        } else {
#pragma unroll
          for (int i = 0; i < kRun; ++i) y[i] = ptx::bf16_lo(q16[from + i]);
        }
      }
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        if constexpr (C::kFmt == WFATTN_CACHE_INT4)  // codes n and n + 4 of a word are a pair
          x[2 * (i / 8) + (i & 3) / 2][2 * (i & 1) + (i >> 2 & 1)] = y[i];
        else
          x[kRun / kE * j + i / kE][i % kE] = y[i];
      }
    }
  }

  // Begins a segment: loads the query rows row0.. of cache head h of sequence b.
  __device__ __forceinline__ void load_q(const Params &p, int b, int h, int row0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < C::kNT; ++nt) {
      const int r = row0 + 8 * nt + g;
      float x[kSteps][kE];
      float top = 0.f, sum = 0.f, mul = 1.f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int e = 0; e < kE; ++e) x[s][e] = 0.f;
      if (r < p.R) {
        const int hg = over_T(p, r), node = r - hg * p.T;
        load_row(p, b * p.qs.b + ((int64_t)h * p.G + hg) * p.qs.h + node * p.qs.s, x);
      }
      if constexpr (C::kKind == kF16) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[s][e]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^14 <= top * mul < 2^15
        const int f = min(max(268 - (int)(__float_as_uint(top) >> 23), 1), 253);
        mul = __uint_as_float((uint32_t)f << 23);
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if constexpr (C::kKind == kTf32) {
          q[nt][s][0] = __float_as_uint(x[s][0]);
          q[nt][s][1] = __float_as_uint(x[s][1]);
        } else if constexpr (C::kKind == kBf16) {
          q[nt][s][0] = ptx::pack_bf16x2(x[s][0], x[s][1]);
          q[nt][s][1] = ptx::pack_bf16x2(x[s][2], x[s][3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[s][e] *= mul;
            sum += x[s][e];
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            q[nt][s][i] = pack_f16x2(x[s][2 * i], x[s][2 * i + 1]);
            if constexpr (kQTerms == 2) {
              const float2 hi = ptx::f16x2_to_f32(q[nt][s][i]);
              q[nt][s][2 + i] = pack_f16x2(x[s][2 * i] - hi.x, x[s][2 * i + 1] - hi.y);
            }
          }
        }
      }
      if constexpr (C::kFmt == WFATTN_CACHE_INT4) {
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      }
      // 1 / mul is a power of two as well
      const float f = p.scale_log2 * __uint_as_float((254u << 23) - __float_as_uint(mul));
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // from query g to queries 2t, 2t + 1
        qf[nt][i] = p.scale_log2;
        if constexpr (C::kKind == kF16) qf[nt][i] = __shfl_sync(0xffffffffu, f, 4 * (2 * t + i));
        if constexpr (C::kFmt == WFATTN_CACHE_INT4)
          qsum[nt][i] = __shfl_sync(0xffffffffu, sum, 4 * (2 * t + i));
        const int rr = row0 + 8 * nt + 2 * t + i;
        const int node = rr - over_T(p, rr) * p.T;
        word[nt][i] = p.tree ? p.tree[b * p.tree_stride + node] : (2ull << node) - 1;
        m[nt][i] = -FLT_MAX;
        l[nt][i] = om[nt][i] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < C::kMt; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][mt][e] = 0.f;
    }
    vinv = __uint_as_float(253u << 23);  // 2^126
    if (C::kScaled && g < 2 * C::kNT) own[4 * g + t] = 0;
  }

  // c = K Q^T of the 16 keys at k.
  __device__ __forceinline__ void scores(uint32_t k, float (&c)[C::kNT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // two chains: even and odd steps, or in split products the leading one and
    // the small ones
    float c2[C::kNT][4];
#pragma unroll
    for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[nt][e] = c2[nt][e] = 0.f;
    if constexpr (C::kKind == kBf16) {
      const int row = lane & 15;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        uint32_t a[4];
        ldmatrix4<false>(k + swizzle<C>(row, 32 * s + 16 * (lane >> 4)), a);
#pragma unroll
        for (int nt = 0; nt < C::kNT; ++nt)
          mma<kBf16>(s & 1 ? c2[nt] : c[nt], a, q[nt][s][0], q[nt][s][1]);
      }
    } else if constexpr (C::kKind == kTf32) {
#pragma unroll
      for (int j = 0; j < C::D / 16; ++j) {
        const uint4 x0 = lds128(k + swizzle<C>(g, 16 * (4 * j + t)));
        const uint4 x1 = lds128(k + swizzle<C>(g + 8, 16 * (4 * j + t)));
        const uint32_t a[2][4] = {{x0.x, x1.x, x0.y, x1.y}, {x0.z, x1.z, x0.w, x1.w}};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) hi[e] = tf32_hi(a[i][e]), lo[e] = tf32_lo(a[i][e]);
#pragma unroll
          for (int nt = 0; nt < C::kNT; ++nt) {
            const uint32_t *qq = q[nt][2 * j + i];
            mma<kTf32>(c2[nt], hi, tf32_lo(qq[0]), tf32_lo(qq[1]));
            mma<kTf32>(c2[nt], lo, tf32_hi(qq[0]), tf32_hi(qq[1]));
            mma<kTf32>(c[nt], hi, tf32_hi(qq[0]), tf32_hi(qq[1]));
          }
        }
      }
    } else {
      auto step = [&](int s, const uint32_t(&a)[4]) {
#pragma unroll
        for (int nt = 0; nt < C::kNT; ++nt) {
          if constexpr (kQTerms == 2) mma<kF16>(c2[nt], a, q[nt][s][2], q[nt][s][3]);
          mma<kF16>(kQTerms == 1 && s & 1 ? c2[nt] : c[nt], a, q[nt][s][0], q[nt][s][1]);
        }
      };
      if constexpr (C::kFmt == WFATTN_CACHE_E4M3) {
#pragma unroll
        for (int j = 0; j < C::D / 64; ++j) {
          const uint4 x0 = lds128(k + swizzle<C>(g, 16 * (t + 4 * j)));
          const uint4 x1 = lds128(k + swizzle<C>(g + 8, 16 * (t + 4 * j)));
          const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a[4] = {ptx::e4m3x2_to_f16x2(w0[i]), ptx::e4m3x2_to_f16x2(w1[i]),
                                   ptx::e4m3x2_to_f16x2(w0[i] >> 16),
                                   ptx::e4m3x2_to_f16x2(w1[i] >> 16)};
            step(4 * j + i, a);
          }
        }
      } else {
        constexpr int kWords = C::D / 32;
        uint32_t w0[kWords], w1[kWords];
        if constexpr (C::D == 64) {
          const uint2 x0 = lds64(k + swizzle<C>(g, 8 * t));
          const uint2 x1 = lds64(k + swizzle<C>(g + 8, 8 * t));
          w0[0] = x0.x, w0[1] = x0.y, w1[0] = x1.x, w1[1] = x1.y;
        } else {
          const uint4 x0 = lds128(k + swizzle<C>(g, 16 * t));
          const uint4 x1 = lds128(k + swizzle<C>(g + 8, 16 * t));
          w0[0] = x0.x, w0[1] = x0.y, w0[2] = x0.z, w0[3] = x0.w;
          w1[0] = x1.x, w1[1] = x1.y, w1[2] = x1.z, w1[3] = x1.w;
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t y0 = w0[i] >> (8 * j), y1 = w1[i] >> (8 * j);
            const uint32_t a[4] = {int4_f16x2<false>(y0), int4_f16x2<false>(y1),
                                   int4_f16x2<true>(y0), int4_f16x2<true>(y1)};
            step(2 * i + j, a);
          }
      }
    }
#pragma unroll
    for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[nt][e] += c2[nt][e];
  }

  // The weights of a tile as the narrow operand of V^T P^T.
  struct Probs {
    uint32_t b[C::kNT][C::kKind == kTf32 ? 1 : kPTerms][2];  // [term][keys 0-7, 8-15]
    float f[C::kNT][C::kKind == kTf32 ? 4 : 1];  // tf32: query g, keys 2t, 2t + 1 of each half
  };
  // pv: weights of keys g, g + 8 (by pairs) for queries 2t, 2t + 1
  __device__ __forceinline__ void operands(const float (&pv)[C::kNT][4], Probs &pr) {
#pragma unroll
    for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = pv[nt][2 * i], y = pv[nt][2 * i + 1];
        if constexpr (C::kKind == kTf32) {
          const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
          const uint32_t hi = movmatrix(__byte_perm(a, b, 0x7632));
          const uint32_t lo = movmatrix(__byte_perm(a, b, 0x5410));
          pr.f[nt][2 * i] = __uint_as_float(__byte_perm(lo, hi, 0x5410));
          pr.f[nt][2 * i + 1] = __uint_as_float(__byte_perm(lo, hi, 0x7632));
        } else if constexpr (C::kKind == kBf16) {
          const uint32_t hi = ptx::pack_bf16x2(x, y);
          pr.b[nt][0][i] = movmatrix(hi);
          pr.b[nt][1][i] =
              movmatrix(ptx::pack_bf16x2(x - ptx::bf16_lo(hi), y - ptx::bf16_hi(hi)));
        } else {
          const uint32_t hi = pack_f16x2(x, y);
          pr.b[nt][0][i] = movmatrix(hi);
          if constexpr (kPTerms == 2) {
            const float2 f = ptx::f16x2_to_f32(hi);
            pr.b[nt][1][i] = movmatrix(pack_f16x2(x - f.x, y - f.y));
          }
        }
      }
  }

  // O^T += V^T P^T over the 16 keys at v.  kTail: what of V is not finite is
  // left out, and the return value tells whether there is any.
  template <bool kTail>
  __device__ __forceinline__ bool values(uint32_t v, const Probs &pr) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    bool odd = false;
    // f32 results: a tile's product is added in f32 arithmetic, so that cut
    // bits do not pile up along the keys
    auto add = [&](int mt, uint32_t(&a)[4]) {
      if constexpr (kTail && C::kFmt != WFATTN_CACHE_INT4) {
        constexpr uint32_t kExp = C::kKind == kBf16 ? 0x7f80u : 0x7c00u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((a[e] & kExp) == kExp) a[e] &= 0xffff0000u, odd = true;
          if ((a[e] >> 16 & kExp) == kExp) a[e] &= 0xffffu, odd = true;
        }
      }
#pragma unroll
      for (int nt = 0; nt < C::kNT; ++nt) {
        if constexpr (C::kF32) {
          float z[4] = {0.f, 0.f, 0.f, 0.f};
          if constexpr (kPTerms == 2) mma<C::kKind>(z, a, pr.b[nt][1][0], pr.b[nt][1][1]);
          mma<C::kKind>(z, a, pr.b[nt][0][0], pr.b[nt][0][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][mt][e] += z[e];
        } else {
          if constexpr (kPTerms == 2)
            mma<C::kKind>(o[nt][mt], a, pr.b[nt][1][0], pr.b[nt][1][1]);
          mma<C::kKind>(o[nt][mt], a, pr.b[nt][0][0], pr.b[nt][0][1]);
        }
      }
    };
    if constexpr (C::kKind == kBf16) {
      const int row = (lane & 7) + 8 * (lane >> 4);
#pragma unroll
      for (int mt = 0; mt < C::kMt; ++mt) {
        uint32_t a[4];
        ldmatrix4<true>(v + swizzle<C>(row, 32 * mt + 16 * (lane >> 3 & 1)), a);
        add(mt, a);
      }
    } else if constexpr (C::kKind == kTf32) {
#pragma unroll
      for (int h = 0; h < C::D / 32; ++h) {
        uint32_t x[4][4];  // keys 2t, 2t + 1 of each half
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 y = lds128(v + swizzle<C>(2 * t + (i & 1) + 8 * (i >> 1), 16 * (g + 8 * h)));
          x[i][0] = y.x, x[i][1] = y.y, x[i][2] = y.z, x[i][3] = y.w;
          if constexpr (kTail) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if ((x[i][e] & 0x7f800000u) == 0x7f800000u) x[i][e] = 0, odd = true;
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t hi[2][4], lo[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t a = x[2 * i + (e >> 1)][2 * j + (e & 1)];
              hi[i][e] = tf32_hi(a), lo[i][e] = tf32_lo(a);
            }
#pragma unroll
          for (int nt = 0; nt < C::kNT; ++nt) {
            float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t p0 = __float_as_uint(pr.f[nt][2 * i]);
              const uint32_t p1 = __float_as_uint(pr.f[nt][2 * i + 1]);
              mma<kTf32>(z, hi[i], tf32_lo(p0), tf32_lo(p1));
              mma<kTf32>(z, lo[i], tf32_hi(p0), tf32_hi(p1));
              mma<kTf32>(z, hi[i], tf32_hi(p0), tf32_hi(p1));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][2 * h + j][e] += z[e];
          }
        }
      }
    } else if constexpr (C::kFmt == WFATTN_CACHE_E4M3) {
      constexpr int kWords = C::D / 32;
      uint32_t x[4][kWords];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 2 * t + (i & 1) + 8 * (i >> 1);
        if constexpr (C::D == 64) {
          const uint2 y = lds64(v + swizzle<C>(row, 8 * g));
          x[i][0] = y.x, x[i][1] = y.y;
        } else {
          const uint4 y = lds128(v + swizzle<C>(row, 16 * g));
          x[i][0] = y.x, x[i][1] = y.y, x[i][2] = y.z, x[i][3] = y.w;
        }
      }
#pragma unroll
      for (int i = 0; i < kWords; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t y0 = __byte_perm(x[0][i], x[1][i], j ? 0x7362 : 0x5140);
          const uint32_t y1 = __byte_perm(x[2][i], x[3][i], j ? 0x7362 : 0x5140);
          uint32_t a[4] = {ptx::e4m3x2_to_f16x2(y0), ptx::e4m3x2_to_f16x2(y0 >> 16),
                           ptx::e4m3x2_to_f16x2(y1), ptx::e4m3x2_to_f16x2(y1 >> 16)};
          add(2 * i + j, a);
        }
    } else {
      constexpr int kWords = C::D / 64;
      uint32_t x[4][kWords];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 2 * t + (i & 1) + 8 * (i >> 1);
        if constexpr (C::D == 64) {
          x[i][0] = lds32(v + swizzle<C>(row, 4 * g));
        } else {
          const uint2 y = lds64(v + swizzle<C>(row, 8 * g));
          x[i][0] = y.x, x[i][1] = y.y;
        }
      }
#pragma unroll
      for (int i = 0; i < kWords; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t y0 = __byte_perm(x[0][i], x[1][i], h ? 0x7632 : 0x5410);
          const uint32_t y1 = __byte_perm(x[2][i], x[3][i], h ? 0x7632 : 0x5410);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t z0 = y0 >> (8 * j), z1 = y1 >> (8 * j);
            uint32_t a[4] = {int4_f16x2<false>(z0), int4_f16x2<true>(z0), int4_f16x2<false>(z1),
                             int4_f16x2<true>(z1)};
            add(4 * i + 2 * h + j, a);
          }
        }
    }
    return odd;
  }

  // What values<true>() left out, where a weight of 0 would have spread it:
  // queries that see its key get it here.  pv: < 0 where the key is not seen.
  __device__ __forceinline__ void not_finite(uint32_t v, const float (&pv)[C::kNT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if constexpr (C::kFmt != WFATTN_CACHE_INT4) {
#pragma unroll 1
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float x = __shfl_sync(0xffffffffu, r < 8 ? pv[nt][i] : pv[nt][2 + i],
                                        4 * (r & 7) + t);
            if (x < 0.f) continue;
#pragma unroll
            for (int mt = 0; mt < C::kMt; ++mt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float y = v_value<C>(v, r, o_index<C>(mt, g, e));
                if (!(fabsf(y) <= FLT_MAX)) o[nt][mt][2 * e + i] += x * y;
              }
          }
    }
  }

  // 2^7 <= top * vinv < 2^8: weights of 2^4 times scales up to 2^11 stay below
  // 2^16, and a weight has all its 11 bits down to 2^-21.
  static __device__ __forceinline__ float vinv_of(float top) {
    const int f = min(max(261 - (int)(__float_as_uint(top) >> 23), 1), 253);
    return __uint_as_float((uint32_t)f << 23);
  }

  // A tail's weights: each query's vinv follows the scales that it sees, and what
  // it does not see has weight 0 whatever its scale.
  __device__ __forceinline__ void tail_weights(const float (&d)[C::kKT][C::kNT][4],
                                               const float (&vs)[C::kKT][2],
                                               float (&pv)[C::kKT][C::kNT][4]) {
#pragma unroll
    for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mine = own_vinv(nt, i), top = 0.f;
#pragma unroll
        for (int j = 0; j < C::kKT; ++j)
#pragma unroll
          for (int e = i; e < 4; e += 2)
            if (d[j][nt][e] != -INFINITY) top = fmaxf(top, fabsf(vs[j][e >> 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const bool change = top * mine > 2048.f;  // the same for all that hold the query
        if (__any_sync(0xffffffffu, change)) {
          const float now = change ? vinv_of(top) : mine, ratio = now / mine;
          mine = now;
#pragma unroll
          for (int mt = 0; mt < C::kMt; ++mt) o[nt][mt][i] *= ratio, o[nt][mt][2 + i] *= ratio;
          if ((threadIdx.x & 31) < 4)
            own[8 * nt + 2 * threadIdx.x % 8 + i] = __float_as_int(now) - __float_as_int(vinv);
          __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < C::kKT; ++j)
#pragma unroll
          for (int e = i; e < 4; e += 2)
            pv[j][nt][e] = d[j][nt][e] == -INFINITY
                               ? 0.f
                               : ptx::ex2_approx(d[j][nt][e]) * (vs[j][e >> 1] * mine);
      }
  }

  // Attends to the 16 kKT keys of rows tr.. of the stage `st`, key0 their
  // position.  kTail: some of them are nodes of the tree, or no keys.
  template <bool kTail>
  __device__ __forceinline__ void group(uint32_t st, int tr, int key0, const Seq &seq) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
    const uint32_t k = st + tr * C::kRowBytes;  // rows 16 apart have the same swizzle
    const uint32_t scales = st + 2 * C::kKBytes + 4 * (tr + g);
    float c[C::kKT][C::kNT][4], vs[C::kKT][2], vm[C::kKT][2];
#pragma unroll
    for (int j = 0; j < C::kKT; ++j) scores(k + 16 * j * C::kRowBytes, c[j]);

    // ---- scales of keys g and g + 8
    if constexpr (C::kScaled) {
#pragma unroll
      for (int j = 0; j < C::kKT; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t at = scales + 4 * (16 * j + 8 * i);
          const uint32_t ks = lds32(at), vw = lds32(at + 4 * C::kKeys);
          // 0, or NaN where the scale is not finite: a score of -inf would hide the key
          if constexpr (C::kFmt == WFATTN_CACHE_E4M3) {
            const float s = __uint_as_float(ks), odd = s - s;
            vs[j][i] = __uint_as_float(vw);
#pragma unroll
            for (int nt = 0; nt < C::kNT; ++nt) {
              c[j][nt][2 * i] = fmaf(c[j][nt][2 * i], s, odd);
              c[j][nt][2 * i + 1] = fmaf(c[j][nt][2 * i + 1], s, odd);
            }
          } else {
            const float s = ptx::bf16_lo(ks), mid = fmaf(8.f, s, ptx::bf16_hi(ks)), odd = s - s;
            vs[j][i] = ptx::bf16_lo(vw);
            vm[j][i] = fmaf(8.f, vs[j][i], ptx::bf16_hi(vw));
#pragma unroll
            for (int nt = 0; nt < C::kNT; ++nt) {
              c[j][nt][2 * i] = fmaf(c[j][nt][2 * i], s, fmaf(mid, qsum[nt][0], odd));
              c[j][nt][2 * i + 1] = fmaf(c[j][nt][2 * i + 1], s, fmaf(mid, qsum[nt][1], odd));
            }
          }
        }
    }

    // ---- weights: 2^(score - m), m raised first where a score is far above it
    float d[C::kKT][C::kNT][4], high = -INFINITY, vtop = 0.f;
#pragma unroll
    for (int j = 0; j < C::kKT; ++j) {
#pragma unroll
      for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          d[j][nt][e] = fmaf(c[j][nt][e], qf[nt][e & 1], -m[nt][e & 1]);
      if constexpr (C::kScaled) vtop = fmaxf(vtop, fmaxf(fabsf(vs[j][0]), fabsf(vs[j][1])));
    }
    if constexpr (kTail) {
#pragma unroll
      for (int j = 0; j < C::kKT; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int node = key0 + 16 * j + 8 * i + g - seq.len;
#pragma unroll
          for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (node >= 0 && (node >= seq.n || !(word[nt][e] >> node & 1)))
                d[j][nt][2 * i + e] = -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < C::kKT; ++j)
#pragma unroll
      for (int nt = 0; nt < C::kNT; ++nt)
        high = fmaxf(high, fmaxf(ptx::fmax3(d[j][nt][0], d[j][nt][1], d[j][nt][2]), d[j][nt][3]));
    bool raise = high > 4.f;
    if constexpr (C::kScaled) raise = raise || (!kTail && vtop * vinv > 2048.f);
    if (__any_sync(0xffffffffu, raise)) {
      float ratio = 1.f;
      if constexpr (C::kScaled && !kTail) {
        float top = vtop;
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        if (top * vinv > 2048.f) {  // the same in the whole warp
          const float now = vinv_of(top);
          ratio = now / vinv;
          vinv = now;
        }
      }
#pragma unroll
      for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = m[nt][i];
#pragma unroll
          for (int j = 0; j < C::kKT; ++j)
#pragma unroll
            for (int e = i; e < 4; e += 2)
              if (d[j][nt][e] != -INFINITY) top = fmaxf(top, c[j][nt][e] * qf[nt][i]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float f = ptx::ex2_approx(m[nt][i] - top);
          m[nt][i] = top;
          l[nt][i] *= f;
          om[nt][i] *= f;
#pragma unroll
          for (int j = 0; j < C::kKT; ++j)
#pragma unroll
            for (int e = i; e < 4; e += 2)
              if (d[j][nt][e] != -INFINITY) d[j][nt][e] = fmaf(c[j][nt][e], qf[nt][i], -top);
#pragma unroll
          for (int mt = 0; mt < C::kMt; ++mt) {
            o[nt][mt][i] *= f * ratio;
            o[nt][mt][2 + i] *= f * ratio;
          }
        }
    }

    float pv[C::kKT][C::kNT][4];
    Probs pr[C::kKT];
#pragma unroll
    for (int j = 0; j < C::kKT; ++j) {
      const float w[2] = {vs[j][0] * vinv, vs[j][1] * vinv};
#pragma unroll
      for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = ptx::ex2_approx(d[j][nt][e]);
          l[nt][e & 1] += x;
          pv[j][nt][e] = C::kScaled ? x * w[e >> 1] : x;
          if constexpr (C::kFmt == WFATTN_CACHE_INT4) {
            float y = x * vm[j][e >> 1];
            if (kTail && d[j][nt][e] == -INFINITY) y = 0.f;  // a scale may be NaN
            om[nt][e & 1] += y;
          }
        }
    }
    if constexpr (C::kScaled && kTail) tail_weights(d, vs, pv);
#pragma unroll
    for (int j = 0; j < C::kKT; ++j) operands(pv[j], pr[j]);
    if constexpr (!kTail) {
#pragma unroll
      for (int j = 0; j < C::kKT; ++j)
        values<false>(k + C::kKBytes + 16 * j * C::kRowBytes, pr[j]);
    } else {
#pragma unroll
      for (int j = 0; j < C::kKT; ++j) {
        const uint32_t v = k + C::kKBytes + 16 * j * C::kRowBytes;
        const bool odd = values<true>(v, pr[j]);
        if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
          for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (d[j][nt][e] == -INFINITY) pv[j][nt][e] = -1.f;
          not_finite(v, pv[j]);
        }
      }
    }
  }
};

// Where the row r of a segment goes, or null: no such row.  `live`: the node
// is no padding.
__device__ __forceinline__ uint8_t *out_row(const Params &p, int64_t b, int64_t h, int r, int n,
                                            int size, bool &live) {
  if (r >= p.R) return nullptr;
  const int hg = over_T(p, r), node = r - hg * p.T;
  live = node < n;
  return p.o + (b * p.os.b + (h * p.G + hg) * p.os.h + node * p.os.s) * size;
}

template <bool kF32>
__device__ __forceinline__ void store_out(uint8_t *row, int d, float x) {
  if constexpr (kF32)
    reinterpret_cast<float *>(row)[d] = x;
  else
    reinterpret_cast<uint16_t *>(row)[d] = (uint16_t)ptx::pack_bf16x2(x, 0.f);
}

// Four values d.. of an output row.
template <bool kF32>
__device__ __forceinline__ void store_out4(const Params &p, uint8_t *row, int d, float4 x) {
  if (p.o_vec && kF32) {
    *reinterpret_cast<float4 *>(row + 4 * d) = x;
  } else if (p.o_vec) {
    *reinterpret_cast<uint2 *>(row + 2 * d) =
        make_uint2(ptx::pack_bf16x2(x.x, x.y), ptx::pack_bf16x2(x.z, x.w));
  } else {
    store_out<kF32>(row, d, x.x);
    store_out<kF32>(row, d + 1, x.y);
    store_out<kF32>(row, d + 2, x.z);
    store_out<kF32>(row, d + 3, x.w);
  }
}

// Adds parts first + begin, first + begin + step, .. up to `last` of values dd.. of
// row r to (m, l, o), eight in flight.  Part c is slot 1 of CTA first, where the
// segment begins, and slot 0 of the others; where there are fewer units than
// CTAs, those without a unit have none.
template <class C>
__device__ __forceinline__ void add_parts(const Params &p, int r, int dd, int first, int last,
                                          int begin, int step, int64_t all, float &m, float &l,
                                          float4 &o) {
  constexpr int kAtOnce = 8;
  const float *ml = p.part + (int64_t)p.ctas * 2 * C::kRows * C::D;
  const bool sparse = all < p.ctas;
#pragma unroll 1
  for (int c0 = first + begin; c0 <= last; c0 += step * kAtOnce) {
    float2 s[kAtOnce];
    float4 z[kAtOnce];
    float top = m;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int c = c0 + j * step;
      s[j] = make_float2(-FLT_MAX, 0.f);
      z[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c <= last && !(sparse && part_of(all, c, p.ctas) == part_of(all, c + 1, p.ctas))) {
        const int64_t at = (int64_t)(c * 2 + (c == first)) * C::kRows + r;
        s[j] = __ldcg(reinterpret_cast<const float2 *>(ml + at * 2));
        z[j] = __ldcg(reinterpret_cast<const float4 *>(p.part + at * C::D + dd));
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) top = fmaxf(top, s[j].x);
    const float f = ptx::ex2_approx(m - top);
    m = top;
    l *= f, o.x *= f, o.y *= f, o.z *= f, o.w *= f;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const float w = ptx::ex2_approx(s[j].x - m);
      l = fmaf(s[j].y, w, l);
      o.x = fmaf(z[j].x, w, o.x), o.y = fmaf(z[j].y, w, o.y);
      o.z = fmaf(z[j].z, w, o.z), o.w = fmaf(z[j].w, w, o.w);
    }
  }
}

// Values dd.. of an output row from its sums.
template <class C>
__device__ __forceinline__ void store_sums(const Params &p, int64_t b, int64_t h, int r, int n,
                                           int dd, float l, float4 o) {
  bool live;
  uint8_t *to = out_row(p, b, h, r, n, C::kF32 ? 4 : 2, live);
  if (!to) return;
  const bool some = live && l != 0.f;
  const float inv = 1.f / l;
  store_out4<C::kF32>(p, to, dd,
                      some ? make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv)
                           : make_float4(0.f, 0.f, 0.f, 0.f));
}

// Counts this CTA's part of a segment, which its threads have written, as
// arrived, and joins the parts if it is the last: of one or two query rows, a
// thread takes a float4 column and every groups-th part, and they meet in `room`
// (3 KB of shared memory).  Not inlined: a CTA comes here twice at most, and the
// loads in flight would cost the main loop its registers.
template <class C>
__device__ __noinline__ void join(const Params &p, int b, int h, int n, int first, int last,
                                  int parts, int64_t all, uint8_t *room) {
  __shared__ int is_last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    is_last = atomicInc(p.arrived + first, parts - 1) == (unsigned)(parts - 1);
    __threadfence();
  }
  __syncthreads();
  if (!is_last) return;
  constexpr int kCols = C::D / 4;
  static_assert(kThreads % (2 * kCols) == 0 && kThreads > 2 * kCols, "whole groups, two at least");
  const int items = p.R * kCols, groups = kThreads / items;
  const int group = threadIdx.x / items, x = threadIdx.x % items;
  const int r = x / kCols, dd = x % kCols * 4;
  float m = -FLT_MAX, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  add_parts<C>(p, r, dd, first, last, group, groups, all, m, l, o);
  float4 *sums = reinterpret_cast<float4 *>(room);
  float2 *mls = reinterpret_cast<float2 *>(room + kThreads * sizeof(float4));
  sums[threadIdx.x] = o;
  mls[threadIdx.x] = make_float2(m, l);
  __syncthreads();
  if (group > 0) return;
  for (int y = 1; y < groups; ++y) m = fmaxf(m, mls[y * items + x].x);
  const float f = ptx::ex2_approx(mls[x].x - m);
  l *= f, o.x *= f, o.y *= f, o.z *= f, o.w *= f;
  for (int y = 1; y < groups; ++y) {
    const float2 s = mls[y * items + x];
    const float4 z = sums[y * items + x];
    const float w = ptx::ex2_approx(s.x - m);
    l = fmaf(s.y, w, l);
    o.x = fmaf(z.x, w, o.x), o.y = fmaf(z.y, w, o.y);
    o.z = fmaf(z.z, w, o.z), o.w = fmaf(z.w, w, o.w);
  }
  store_sums<C>(p, b, h, r, n, dd, l, o);
}

template <class C>
__global__ void __launch_bounds__(kThreads, C::kCtas) 
    tree_decode_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int own[kWarps][8 * C::kNT];  // of Warp
  float *stats = reinterpret_cast<float *>(smem + C::kStages * C::kStage);
  const uint32_t ring = ptx::smem_u32(smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rw = warp / C::kKW, kw = warp % C::kKW;

  int64_t begin, end, all;
  Cursor<C::kKeys> cur = share<C::kKeys>(p, begin, end, all), ahead = cur;
  const int64_t units = end - begin;
  if (p.apart && threadIdx.x == 0) p.split[blockIdx.x].b = -1;
  if (units <= 0) return;

  // Who loads what of a unit: where every warp reads keys of its own, each warp
  // loads those and waits for nobody else; otherwise the CTA loads together.
  // A loader's 16-byte pieces of K (and V) lie kStep apart, in kRuns runs.
  constexpr bool kOwn = C::kRW == 1;
  constexpr int kLoaders = kOwn ? 32 : kThreads, kStep = 16 * kLoaders;
  constexpr int kRuns = kOwn ? C::kGroups : 1;  // a group's rows, kApart rows from the next
  constexpr int kRunRows = kOwn ? 16 * C::kKT : C::kKeys, kApart = 16 * C::kKT * C::kKW;
  constexpr int kPieces = kRunRows * C::kRowBytes / kStep;
  static_assert(kPieces * kStep == kRunRows * C::kRowBytes, "whole pieces");
  const int loader = kOwn ? lane : threadIdx.x;
  const int first = kOwn ? kw * kRunRows : 0;        // row
  const int row0 = loader * 16 / C::kRowBytes;       // in the first kStep bytes of a run
  const uint32_t dst0 = ring + first * C::kRowBytes + swizzle<C>(row0, loader * 16 % C::kRowBytes);
  // `first` and runs are multiples of 16 rows, so the swizzle is row0's and the step's
  auto place = [&](int run, int j) {
    return (dst0 ^ swizzle_bits<C>(j * kStep / C::kRowBytes)) + j * kStep +
           run * kApart * C::kRowBytes;
  };
  const uint8_t *k_at, *v_at;  // the unit fetched next, from this thread's first piece
  const uint8_t *ks_at = nullptr, *vs_at = nullptr;
  auto aim = [&]() {
    const int64_t row = ahead.b * p.c.sb + ahead.h * p.c.sh + (int64_t)ahead.u * C::kKeys + first;
    k_at = p.c.k + row * C::kRowBytes + loader * 16;
    v_at = p.c.v + row * C::kRowBytes + loader * 16;
    if constexpr (C::kScaled) {
      ks_at = p.c.k_scale + row * 4;
      vs_at = p.c.v_scale + row * 4;
    }
  };
  aim();
  int64_t to_fetch = units;
  uint32_t fetch_st = 0;  // stage filled next
  auto fetch = [&]() {
    if (to_fetch > 0) {
      --to_fetch;
      const int live = ahead.s.total - ahead.u * C::kKeys - first;  // rows from `first` on
      const uint32_t st = fetch_st;
      if (live >= kRunRows + (kRuns - 1) * kApart) {
#pragma unroll
        for (int r = 0; r < kRuns; ++r)
#pragma unroll
          for (int j = 0; j < kPieces; ++j) {
            const int off = j * kStep + r * kApart * C::kRowBytes;
            cp_async16(st + place(r, j), k_at + off);
            cp_async16(st + place(r, j) + C::kKBytes, v_at + off);
          }
      } else {
#pragma unroll
        for (int r = 0; r < kRuns; ++r)
#pragma unroll
          for (int j = 0; j < kPieces; ++j) {
            const int off = j * kStep + r * kApart * C::kRowBytes;
            const bool use = row0 + j * (kStep / C::kRowBytes) + r * kApart < live;
            cp_async16(st + place(r, j), use ? k_at + off : p.c.k, use);
            cp_async16(st + place(r, j) + C::kKBytes, use ? v_at + off : p.c.v, use);
          }
      }
      if constexpr (C::kScaled) {
        // a run's scales of K, then those of V
        constexpr int kWords = 2 * kRunRows / kLoaders;
#pragma unroll
        for (int r = 0; r < kRuns; ++r)
#pragma unroll
          for (int j = 0; j < kWords; ++j) {
            const int i = loader + j * kLoaders;
            const int row = (i % kRunRows) + r * kApart;
            const uint8_t *from = i < kRunRows ? ks_at : vs_at;
            const bool use = row < live;
            cp_async4(ring + st + 2 * C::kKBytes + 4 * (first + row) +
                          (i < kRunRows ? 0 : 4 * C::kKeys),
                      use ? from + 4 * row : p.c.k_scale, use);
          }
      }
      fetch_st = fetch_st == (C::kStages - 1) * C::kStage ? 0 : fetch_st + C::kStage;
      if (ahead.next(p)) {
        if (to_fetch > 0) aim();
      } else {
        k_at += C::kKBytes;
        v_at += C::kKBytes;
        if constexpr (C::kScaled) {
          ks_at += 4 * C::kKeys;
          vs_at += 4 * C::kKeys;
        }
      }
    }
    cp_async_commit();
  };

#pragma unroll 1
  for (int i = 0; i < C::kStages - 1; ++i) fetch();
  bool headed = cur.u == 0;  // the segment begins in this CTA
  uint32_t st = 0;
  int64_t i = 0;
#pragma unroll 1
  while (i < units) {  // a segment, or the part of it in this share
    Warp<C> w;
    w.own = own[warp];
    w.load_q(p, cur.b, cur.h, cur.tile * C::kRows + rw * 8 * C::kNT);
    bool done;
#pragma unroll 1
    while (true) {  // a unit
      cp_async_wait<C::kStages - 2>();
      // the unit is here, and the stage refilled next has been read
      if constexpr (kOwn)
        __syncwarp();
      else
        __syncthreads();
      fetch();
      const int key0 = cur.u * C::kKeys;
#pragma unroll 1
      for (int j = 0; j < C::kGroups; ++j) {
        const int tr = 16 * C::kKT * (kw + C::kKW * j);
        if (tr >= cur.s.total - key0) break;
        if (key0 + tr + 16 * C::kKT > cur.s.len)
          w.template group<true>(ring + st, tr, key0 + tr, cur.s);
        else
          w.template group<false>(ring + st, tr, key0 + tr, cur.s);
      }
      done = cur.u + 1 == cur.s.units;
      if (done || i + 1 == units) break;
      ++i;
      ++cur.u;
      st = st == (C::kStages - 1) * C::kStage ? 0 : st + C::kStage;
    }

    const bool whole = done && headed;
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          w.l[nt][e] += __shfl_xor_sync(0xffffffffu, w.l[nt][e], x);
          if constexpr (C::kFmt == WFATTN_CACHE_INT4)
            w.om[nt][e] += __shfl_xor_sync(0xffffffffu, w.om[nt][e], x);
        }
        if constexpr (C::kScaled) {
          const float back = 1.f / w.own_vinv(nt, e);
#pragma unroll
          for (int mt = 0; mt < C::kMt; ++mt) {
            w.o[nt][mt][e] = w.o[nt][mt][e] * back + w.om[nt][e];
            w.o[nt][mt][2 + e] = w.o[nt][mt][2 + e] * back + w.om[nt][e];
          }
        }
      }
    const int slot = headed ? 1 : 0;
    const int rows = min(C::kRows, p.R - cur.tile * C::kRows);  // that there are
    float *part = p.part + (int64_t)(blockIdx.x * 2 + slot) * C::kRows * C::D;
    float *part_ml = p.part + (int64_t)p.ctas * 2 * C::kRows * C::D +
                     (int64_t)(blockIdx.x * 2 + slot) * C::kRows * 2;
    // The warps' sums meet in the stage just read: rows of O, and beside them
    // maximum and sum.  (With all the keys in one warp this only turns the
    // fragments into rows.)
    __syncthreads();
    float *sums = reinterpret_cast<float *>(smem + st);
#pragma unroll
    for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = warp * 8 * C::kNT + 8 * nt + 2 * t + e;
#pragma unroll
        for (int mt = 0; mt < C::kMt; ++mt) {
          if constexpr (C::kKind == kBf16) {
#pragma unroll
            for (int y = 0; y < 2; ++y)
              sums[sum_index<C>(r, o_index<C>(mt, g, y))] = w.o[nt][mt][2 * y + e];
          } else {  // values d and d + 1
            *reinterpret_cast<float2 *>(sums + sum_index<C>(r, o_index<C>(mt, g, 0))) =
                make_float2(w.o[nt][mt][e], w.o[nt][mt][2 + e]);
          }
        }
        if (g == 0) *reinterpret_cast<float2 *>(stats + r * 2) = make_float2(w.m[nt][e], w.l[nt][e]);
      }
    __syncthreads();
#pragma unroll 1
    for (int x = threadIdx.x; x < rows * (C::D / 4); x += kThreads) {
      const int r = x / (C::D / 4), dd = x % (C::D / 4) * 4;
      const int at0 = r / (8 * C::kNT) * C::kKW * 8 * C::kNT + r % (8 * C::kNT);
      float2 ml[C::kKW];
      float m = -FLT_MAX, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int y = 0; y < C::kKW; ++y) {
        ml[y] = *reinterpret_cast<const float2 *>(stats + (at0 + y * 8 * C::kNT) * 2);
        m = fmaxf(m, ml[y].x);
      }
#pragma unroll
      for (int y = 0; y < C::kKW; ++y) {
        const float f = ptx::ex2_approx(ml[y].x - m);
        const float4 z = *reinterpret_cast<const float4 *>(
            sums + sum_index<C>(at0 + y * 8 * C::kNT, dd));
        l = fmaf(ml[y].y, f, l);
        o.x = fmaf(z.x, f, o.x), o.y = fmaf(z.y, f, o.y);
        o.z = fmaf(z.z, f, o.z), o.w = fmaf(z.w, f, o.w);
      }
      if (whole) {
        store_sums<C>(p, cur.b, cur.h, cur.tile * C::kRows + r, cur.s.n, dd, l, o);
      } else {
        *reinterpret_cast<float4 *>(part + r * C::D + dd) = o;
        if (dd == 0) *reinterpret_cast<float2 *>(part_ml + 2 * r) = make_float2(m, l);
      }
    }
    constexpr bool kJoins = C::kRows == 8;  // the configuration of one or two query rows
    if (!kJoins || p.apart) {
      if (!done && headed && threadIdx.x == 0)
        p.split[blockIdx.x] = split_of(p, cur, begin + i - cur.u, all);
    } else if (!whole) {
      if constexpr (kJoins) {
        // CTAs without units are passed over; there are none, or no CTA has two
        const int64_t s0 = begin + i - cur.u;
        const int first_cta =
            headed ? (int)blockIdx.x : (int)(((s0 + 1) * p.ctas - 1) / all);
        const int last_cta = split_of(p, cur, s0, all).last;
        const int parts = min(last_cta - first_cta + 1, cur.s.units);
        join<C>(p, cur.b, cur.h, cur.s.n, first_cta, last_cta, parts, all, smem + st);
      }
    }
    // the stage may be refilled once all have read it (with common loads the
    // next unit's barrier says so)
    if constexpr (kOwn) __syncthreads();
    headed = true;
    st = st == (C::kStages - 1) * C::kStage ? 0 : st + C::kStage;
    cur.next(p);
    ++i;
  }
  cp_async_wait<0>();
}

// ------------------------------------------------------------------ launch

template <class C>
size_t workspace_bytes() {
  static_assert(C::kCtas * kMaxSms <= kCounters, "a counter a CTA");
  static_assert(C::kCtas * kMaxSms * sizeof(Split) % 16 == 0, "parts are read 16 bytes at a time");
  return kCounters * sizeof(unsigned int) + kMaxSms * C::kCtas * sizeof(Split) +
         (size_t)kMaxSms * C::kCtas * 2 * C::kRows * (C::D + 2) * sizeof(float);
}

// Joins the parts of the segments that more than one CTA worked on.  A thread takes
// four values of a row and, where there are few rows, every kth of its parts: all
// the loads there are should be in flight at once, as a round of them takes a
// microsecond.  One 15-node tree over 4,000 bf16 rows, 8 heads of 37 parts each: a
// call takes 25 us, against 43 with four rows a thread one after the other and
// all of a row's parts; with one cache head of 63 parts 17 against 63.
constexpr int kJoinThreads = 256, kJoinBlocks = 3 * kMaxSms;

template <class C>
__global__ void __launch_bounds__(kJoinThreads, 3)
    tree_join_kernel(const __grid_constant__ Params p) {
  constexpr int kCols = C::D / 4, kMost = kJoinThreads / kCols;
  __shared__ int heads[kMaxSms * C::kCtas];  // CTAs where a segment that goes on begins
  __shared__ int counts[kJoinThreads / 32];
  __shared__ float4 sums[kJoinThreads];
  __shared__ float2 mls[kJoinThreads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // launched before the parts are there (launch_join)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // after a wait ran out the records may be another call's
  if (C::kWide && __syncthreads_or(ptx::timeout_flagged(p.status))) return;
  constexpr int kTimes = (kMaxSms * C::kCtas + kJoinThreads - 1) / kJoinThreads;
  bool goes_on[kTimes];
#pragma unroll
  for (int t = 0; t < kTimes; ++t) {
    const int x = t * kJoinThreads + tid;
    goes_on[t] = x < p.ctas && p.split[x].b >= 0;
  }
  int segments = 0;
#pragma unroll
  for (int t = 0; t < kTimes; ++t) {  // in order, the same in every block
    const bool live = goes_on[t];
    const unsigned mask = __ballot_sync(0xffffffffu, live);
    if (lane == 0) counts[warp] = __popc(mask);
    __syncthreads();
    int at = segments + __popc(mask & ((1u << lane) - 1));
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) {
      if (w < warp) at += counts[w];
      segments += counts[w];
    }
    if (live) heads[at] = t * kJoinThreads + tid;
    __syncthreads();
  }
  const int rows = min(C::kRows, p.R), total = segments * rows;
  int k = 1;  // threads that share a row's parts
  while (k < kMost && total * kCols * k * 2 <= (int)gridDim.x * kJoinThreads) k *= 2;
  const int teams = kMost / k, team = tid / (kCols * k), group = tid / kCols % k;
  const int dd = tid % kCols * 4;
#pragma unroll 1
  for (int i0 = blockIdx.x * teams; i0 < total; i0 += gridDim.x * teams) {
    const int i = i0 + team, head = heads[min(i, total - 1) / rows], r = i % rows;
    const Split s = p.split[head];
    const bool live = i < total && s.tile * C::kRows + r < p.R;
    const int n = sequence<C::kKeys>(p, s.b, false).n;
    float m = -FLT_MAX, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) add_parts<C>(p, r, dd, head, s.last, group, k, s.all, m, l, o);
    if (k > 1) {
      sums[tid] = o;
      mls[tid] = make_float2(m, l);
      __syncthreads();
      if (group == 0) {
        const float own = m;
        for (int y = 1; y < k; ++y) m = fmaxf(m, mls[tid + y * kCols].x);
        const float f = ptx::ex2_approx(own - m);
        l *= f, o.x *= f, o.y *= f, o.z *= f, o.w *= f;
        for (int y = 1; y < k; ++y) {
          const float2 t = mls[tid + y * kCols];
          const float4 z = sums[tid + y * kCols];
          const float w = ptx::ex2_approx(t.x - m);
          l = fmaf(t.y, w, l);
          o.x = fmaf(z.x, w, o.x), o.y = fmaf(z.y, w, o.y);
          o.z = fmaf(z.z, w, o.z), o.w = fmaf(z.w, w, o.w);
        }
      }
      __syncthreads();
    }
    if (live && group == 0)
      store_sums<C>(p, s.b, s.h, s.tile * C::kRows + r, n, dd, l, o);
  }
}

template <class C>
cudaError_t launch_join(const Params &p, cudaStream_t stream) {
  const cudaError_t err = cudaGetLastError();  // of the launch before
  // segments of at most kShort units are dealt whole
  if (err != cudaSuccess || p.c.L <= kShort * C::kKeys) return err;
  const int rows = p.R < C::kRows ? p.R : C::kRows;
  // a segment a CTA at most, and up to all of a block for one of its rows
  const int blocks = p.ctas * rows < kJoinBlocks ? p.ctas * rows : kJoinBlocks;
  // It may be launched as the blocks before it end, and waits for what they wrote
  // itself: 1.5 us less a call (2 to 3%) of those that a host launches one by one.
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(kJoinThreads);
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, tree_join_kernel<C>, p);
}

// The parameters that go with the configuration.
template <class C>
void prepare(Params &p, void *workspace, const DeviceInfo &dev) {
  p.RT = (p.R + C::kRows - 1) / C::kRows;
  p.over_T = (uint32_t)(((uint64_t(1) << 32) + p.T - 1) / p.T);  // not used for T = 1
  const uintptr_t q16 = reinterpret_cast<uintptr_t>(p.q), o16 = reinterpret_cast<uintptr_t>(p.o);
  constexpr int kVec = C::kF32 ? 4 : 8;  // values in 16 bytes
  p.q_vec = q16 % 16 == 0 && p.qs.b % kVec == 0 && p.qs.h % kVec == 0 && p.qs.s % kVec == 0;
  p.o_vec = o16 % 16 == 0 && p.os.b % kVec == 0 && p.os.h % kVec == 0 && p.os.s % kVec == 0;
  p.apart = p.R > 2;
  const int64_t segs = p.c.B * p.c.H * p.RT;
  const int64_t units = (p.c.L + C::kKeys - 1) / C::kKeys;  // of a segment, at most
  const int64_t most = (dev.sm_count < kMaxSms ? dev.sm_count : kMaxSms) * C::kCtas;
  p.ctas = (int)imin64(most, units > most ? most : units * imin64(segs, most));
  p.arrived = static_cast<unsigned int *>(workspace);
  p.split = reinterpret_cast<Split *>(p.arrived + kCounters);
  p.part = reinterpret_cast<float *>(p.split + kMaxSms * C::kCtas);
}

template <class C>
cudaError_t launch(Params p, void *workspace, const DeviceInfo &dev, cudaStream_t stream) {
  static_assert(C::kStage >= 24 * kThreads, "room to join in");
  prepare<C>(p, workspace, dev);
  const cudaError_t err = ensure_smem_attr(
      reinterpret_cast<const void *>(tree_decode_kernel<C>), C::kSmem, dev.device);
  if (err != cudaSuccess) return err;
  tree_decode_kernel<C><<<p.ctas, kThreads, C::kSmem, stream>>>(p);
  if (C::kRows == 8 && !p.apart) return cudaGetLastError();
  return launch_join<C>(p, stream);
}

}  // namespace tree
}  // namespace wfattn
