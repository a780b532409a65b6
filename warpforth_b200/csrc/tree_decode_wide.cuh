// tree_decode_wide.cuh -- tree_decode for many query rows a cache head: the
// products on tcgen05 tensor cores.
//
// A CTA takes up to 128 query rows of one cache head (one TMEM lane, and one
// thread or two, a row) and walks its keys in units of 64:
//
//   S [128 x 64]   = Q [128 x D] K^T         both operands in shared memory
//   O [128 x D]   += P [128 x 64] V          P in tensor memory
//
// K and V lie in shared memory as 16-bit rows in the 128-byte swizzle that the
// operands have, K along a row and V across rows.  bf16 rows arrive there by
// cp.async; the codes of e4m3 and int4 rows come through registers, a unit
// ahead, and are written as f16 (exactly; int4 as u - 8).  Scales, weights, lazy
// maximum and the split of work are those of tree_decode.cuh; bf16 weights take
// two products (two terms).
//
// Warps 0-3 (4-bit rows: 0-7, half a row's keys a thread) turn scores into
// weights, the next two bring the rows of the units, one issues Q K^T and the last
// P V (a product leaves a warp every 75 clocks or so, which one warp's other work
// would add to).  K and V have two buffers, and so have S and P, which share
// theirs (a thread, or both of a row, has read S before it writes P): while the
// weights of unit i are made, Q K^T of i + 1 is done and the rows of i + 2 follow
// P V of i.  TMEM columns: twice 64 for S and P, 64 or 128 for O; 256 a CTA, two
// CTAs an SM.
//
// With more than 128 query rows a cache head the tiles are segments of their own,
// and each reads and converts the keys again.
//
// Measured: 61-node trees of 4 query heads a cache head over two e4m3 caches of
// 65,000 and 131,000 keys, 8 heads of 128: 412 us, 476 TFLOP/s.  A unit takes a
// CTA about 4,000 clocks; rows are placed in 1,350, S is there 1,500 after Q K^T
// begins, weights take 2,400 and P V 840.  No one of them is the bound: without
// weights it would be 286 us, without conversion 349, with half the products 390.
// 15-node trees, 16 sequences, 40,134 keys of each of 8 heads: 65 us (bf16), 70 (4
// bits), 82 (e4m3).
//
// Every wait has a limit.  After one that runs out the warps that make weights
// go on to the end without waiting; the two of a row meet as often as ever.
#pragma once

#include <type_traits>

#include "tree_decode.cuh"

namespace wfattn {
namespace tree {

constexpr int kLoaders = 64;

template <int kFmt_, int D_>
struct WideCfg {
  static constexpr int kFmt = kFmt_, D = D_, kRows = 128, kKeys = 64, kCtas = 2;
  static constexpr bool kF32 = false, kWide = true;
  static constexpr bool kBf16Rows = kFmt == WFATTN_CACHE_BF16;
  static constexpr bool kScaled = !kBf16Rows;
  static constexpr int kRowBytes = CacheRow<kFmt, D>::kBytes;
  // Threads of a query row.  4-bit rows take two, as their minima make the weights
  // dearer: 15-node trees, 4 query heads on 8, 70 us against 80 (64 values a row: 55
  // against 57); 61-node trees over 196,000 keys 398 against 403 (319 against 286).
  // The others have nothing from it, or lose by 80 registers a thread: bf16 67 us
  // both ways, e4m3 97 against 83.
  static constexpr int kHalves = kFmt == WFATTN_CACHE_INT4 ? 2 : 1;
  static constexpr int kWeighers = kHalves * kThreads, kWideThreads = kWeighers + kThreads;
  static constexpr int kMine = kKeys / kHalves, kDims = D / kHalves;  // of a thread's row
  static constexpr int kSlabs = D / 64;               // 128-byte wide slabs of an operand
  static constexpr int kSlab = kKeys * 128;           // bytes of a slab of K or V
  static constexpr int kQSlab = kRows * 128;
  static constexpr int kBuf = 2 * kSlabs * kSlab;     // K and V of a unit
  static constexpr int kPieces = kKeys * kRowBytes / 16 / kLoaders;  // of K (and V) a loader
  static constexpr int kWork = kSlabs * kQSlab + 2 * kBuf;
  static constexpr int kSmem = kWork + 1024;          // and room to align
  static constexpr uint32_t kColS = 0, kColO = 128, kCols = 256;  // P: as S; 64 a buffer
  static_assert(kKeys == kLoaders, "a loader brings a row's scales");
  static_assert(kSmem <= (227 / kCtas - 3) * 1024, "two CTAs an SM");
};

__device__ __forceinline__ uint32_t idesc_wide(bool bf16, int n, bool b_mn) {
  // M 128, f32 accumulation; formats f16 (0) or bf16 (1)
  return ptx::idesc_bf16_f32(128, n, 0, b_mn ? 1 : 0) & (bf16 ? ~0u : ~((1u << 7) | (1u << 10)));
}

// Byte offset of the 16-byte piece c (8 values) of row r in an operand whose
// slabs have `slab` bytes.
__device__ __forceinline__ uint32_t piece(int r, int c, int slab) {
  return (c >> 3) * slab + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// int4 rows are unpacked as pairs of codes n, n + 4 of a word: value `v` of a
// row's eight is at place `i`.
__device__ __forceinline__ constexpr int int4_place(int v) {
  return 2 * (v & 3) + (v >> 2);
}

__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

// Products and commits issued by a whole warp in step, lane `leader` doing it:
// with the branch inside the instruction's predicate the operands stay in
// uniform registers, and a product leaves every few tens of clocks instead of
// every 200 from a branch that one thread takes.
__device__ __forceinline__ void mma_ss_warp(uint32_t leader, uint32_t d, uint64_t a, uint64_t b,
                                            uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 q, %0, 0;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], %2, %3, %4, p;\n\t}" ::"r"(leader),
      "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts_warp(uint32_t leader, uint32_t d, uint32_t a, uint64_t b,
                                            uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 q, %0, 0;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], %3, %4, p;\n\t}" ::"r"(leader),
      "r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_warp(uint32_t leader, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %0, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(
          leader),
      "r"(bar)
      : "memory");
}

// 16 consecutive TMEM columns of this thread's lane -> registers.
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}

// A value of V in memory, unscaled; used where a row is not finite.
template <class C>
__device__ __forceinline__ float v_in_memory(const uint8_t *row, int d) {
  if constexpr (C::kBf16Rows) return ptx::bf16_lo(reinterpret_cast<const uint16_t *>(row)[d]);
  return ptx::f16x2_to_f32(ptx::e4m3x2_to_f16x2(row[d])).x;
}

// The other half's value of a row's pair of threads (`at` and `other` are their
// places, `pair` their two warps' barrier).  Two sets of places take turns: one
// is written again after the other's barrier, when it has been read.
__device__ __forceinline__ float swap_halves(float x, float *at, const float *other, int pair) {
  *at = x;
  asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
  return *other;
}

// Keys of a unit that a query with this word does not see; key k is node k - at of
// n: bits of the word, or before the tree.
__device__ __forceinline__ uint64_t hidden_keys(int at, int n, uint64_t word) {  // at <= 63
  const uint64_t nodes = n >= 64 ? ~uint64_t(0) : (uint64_t(1) << n) - 1;
  const uint64_t seen = word & nodes;
  return at >= 0 ? ~(at > 0 ? seen << at | ((uint64_t(1) << at) - 1) : seen)
                 : ~(at > -64 ? seen >> -at : 0);
}

// The largest of a thread's scales that its query sees: one that it does not see
// has to leave its weights their bits.  Not inlined: tails alone come here, and
// the rest would be short of registers.
template <class C>
__device__ __noinline__ float seen_top(int at, int n, int half, uint64_t word,
                                       const float *v_scale) {
  const uint64_t hidden = hidden_keys(at, n, word) >> C::kMine * half;
  float top = 0.f;
#pragma unroll 4
  for (int k = 0; k < C::kMine; ++k)
    if (!(hidden >> k & 1)) top = fmaxf(top, fabsf(v_scale[k]));
  return top;
}

// A thread's keys of its row of S, C::kMine * half and on, to weights in tensor
// memory; sp is the row's.  Maximum, sum and (int4) the sum of weights times
// minima go on in m, which both halves know, and l and om, which are this half's.
// swap() gives the other half's value: its thread has read S when it returns, and
// P may take its place.  wait_o() waits for the products added to O so far, and is
// called where O is changed, C::kDims columns by each.
template <class C, bool kTail, class Swap, class Wait>
__device__ __forceinline__ void weigh(const Params &p, const Cursor<C::kKeys> &cur, int half,
                                      uint32_t row_tmem, uint32_t sp, int key0, bool odd,
                                      uint64_t word, float qf, float qsum, const float *k_scale,
                                      const float *k_mid, const float *v_scale, const float *v_mid,
                                      float vtop, bool first, float &m, float &l, float &om,
                                      float &vinv, Swap swap, Wait wait_o) {
  constexpr int kMine = C::kMine;
  if constexpr (kTail && C::kScaled) {
    if (C::kHalves == 2 || __any_sync(0xffffffffu, vtop * vinv > 2048.f)) {
      vtop = seen_top<C>(cur.s.len - key0, cur.s.n, half, word, v_scale);
      if constexpr (C::kHalves == 2) vtop = fmaxf(vtop, swap(vtop));
    }
  }
  uint32_t s[kMine];
  if constexpr (kMine == 64)
    ptx::tmem_ld_32x32b_x64(sp, s);
  else
    ptx::tmem_ld32(sp + kMine * half, s);
  ptx::tmem_wait_ld();
  // ---- scores before qf, which is positive
  const uint64_t qsum2 = ptx::f2_pack(qsum, qsum);
  if constexpr (C::kScaled) {
#pragma unroll
    for (int k = 0; k < kMine; k += 4) {
      const ulonglong2 ks = *reinterpret_cast<const ulonglong2 *>(k_scale + k);
      uint64_t y0 = ptx::f2_pack(__uint_as_float(s[k]), __uint_as_float(s[k + 1]));
      uint64_t y1 = ptx::f2_pack(__uint_as_float(s[k + 2]), __uint_as_float(s[k + 3]));
      if constexpr (C::kFmt == WFATTN_CACHE_INT4) {
        const ulonglong2 mid = *reinterpret_cast<const ulonglong2 *>(k_mid + k);
        y0 = ptx::f2_fma(y0, ks.x, ptx::f2_mul(mid.x, qsum2));
        y1 = ptx::f2_fma(y1, ks.y, ptx::f2_mul(mid.y, qsum2));
      } else {
        y0 = ptx::f2_mul(y0, ks.x);
        y1 = ptx::f2_mul(y1, ks.y);
      }
      float x[4];
      ptx::f2_unpack(y0, x[0], x[1]);
      ptx::f2_unpack(y1, x[2], x[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[k + e] = __float_as_uint(x[e]);
    }
  }
  uint64_t hidden = 0;  // keys of the unit this row does not see
  std::conditional_t<kMine == 64, uint64_t, uint32_t> mine = 0;  // of this thread's
  if constexpr (kTail) {
    hidden = hidden_keys(cur.s.len - key0, cur.s.n, word);
    mine = kMine == 64 ? hidden : hidden >> 32 * half;
#pragma unroll
    for (int k = 0; k < kMine; ++k)
      if (mine >> k & 1) s[k] = 0xff800000u;
  }
  float high4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int k = 0; k < kMine; k += 2)
    high4[k / 2 % 4] =
        ptx::fmax3(high4[k / 2 % 4], __uint_as_float(s[k]), __uint_as_float(s[k + 1]));
  float high = fmaxf(fmaxf(high4[0], high4[1]), fmaxf(high4[2], high4[3]));
  if constexpr (C::kHalves == 2) high = fmaxf(high, swap(high));
  if (__any_sync(0xffffffffu, fmaf(high, qf, -m) > 4.f || vtop * vinv > 2048.f)) {
    float ratio = 1.f;
    if (C::kScaled && vtop * vinv > 2048.f) {
      const int f = min(max(261 - (int)(__float_as_uint(vtop) >> 23), 1), 253);
      const float now = __uint_as_float((uint32_t)f << 23);
      ratio = now / vinv;
      vinv = now;
    }
    const float top = fmaxf(m, high * qf);
    const float f = ptx::ex2_approx(m - top);
    m = top;
    l *= f;
    om *= f;
    if (!first) {
      wait_o();
#pragma unroll 1
      for (int c = C::kDims * half; c < C::kDims * (half + 1); c += 16) {
        uint32_t o[16];
        tmem_ld16(row_tmem + C::kColO + c, o);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e)
          o[e] = __float_as_uint(__uint_as_float(o[e]) * (f * ratio));
        ptx::tmem_st16(row_tmem + C::kColO + c, o);
      }
    }
  }
  const uint64_t qf2 = ptx::f2_pack(qf, qf), m2 = ptx::f2_pack(-m, -m);
  const uint64_t vinv2 = ptx::f2_pack(vinv, vinv);
  uint64_t l2[2] = {0, 0}, om2[2] = {0, 0};
#pragma unroll
  for (int part = 0; part < kMine / 32; ++part) {  // 16 registers of weights at a time
    uint32_t hi[16], lo[C::kBf16Rows ? 16 : 1];
#pragma unroll
    for (int k = 32 * part; k < 32 * part + 32; k += 4) {
      ulonglong2 vs = {0, 0}, mid = {0, 0};
      if constexpr (C::kScaled) vs = *reinterpret_cast<const ulonglong2 *>(v_scale + k);
      if constexpr (C::kFmt == WFATTN_CACHE_INT4)
        mid = *reinterpret_cast<const ulonglong2 *>(v_mid + k);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int kk = k + 2 * e;
        float a, b;
        ptx::f2_unpack(
            ptx::f2_fma(ptx::f2_pack(__uint_as_float(s[kk]), __uint_as_float(s[kk + 1])), qf2, m2),
            a, b);
        a = ptx::ex2_approx(a);
        b = ptx::ex2_approx(b);
        const uint64_t w = ptx::f2_pack(a, b);
        l2[e] = ptx::f2_add(l2[e], w);
        const bool hide_a = kTail && (mine >> kk & 1), hide_b = kTail && (mine >> kk & 2);
        const int to = (kk - 32 * part) / 2;
        if constexpr (C::kScaled) {
          uint64_t vm = e ? mid.y : mid.x;
          if constexpr (C::kFmt == WFATTN_CACHE_INT4) {
            if constexpr (kTail) {  // a scale may be NaN
              float x, y;
              ptx::f2_unpack(vm, x, y);
              vm = ptx::f2_pack(hide_a ? 0.f : x, hide_b ? 0.f : y);
            }
            om2[e] = ptx::f2_fma(w, vm, om2[e]);
          }
          ptx::f2_unpack(ptx::f2_mul(w, ptx::f2_mul(e ? vs.y : vs.x, vinv2)), a, b);
          if (hide_a) a = 0.f;
          if (hide_b) b = 0.f;
          hi[to] = pack_f16x2(a, b);
        } else {
          hi[to] = ptx::pack_bf16x2(a, b);
          lo[to] = ptx::pack_bf16x2(a - ptx::bf16_lo(hi[to]), b - ptx::bf16_hi(hi[to]));
        }
      }
    }
    // S is read: P takes its place
    const uint32_t to = sp + kMine / 2 * half + 16 * part;
    ptx::tmem_st16(to, hi);
    if constexpr (C::kBf16Rows) ptx::tmem_st16(to + 32, lo);
  }
  float a, b;
  ptx::f2_unpack(ptx::f2_add(l2[0], l2[1]), a, b);
  l += a + b;
  if constexpr (C::kFmt == WFATTN_CACHE_INT4) {
    ptx::f2_unpack(ptx::f2_add(om2[0], om2[1]), a, b);
    om += a + b;
  }
  if constexpr (kTail && C::kFmt != WFATTN_CACHE_INT4) {
    if (odd) {
      // What is not finite in V was put to zero in the operand, where a weight
      // of 0 would spread it: rows that see its key get it here.
      const uint8_t *v =
          p.c.v + (cur.b * p.c.sb + cur.h * p.c.sh + (int64_t)key0) * C::kRowBytes;
      const int keys = min(64, cur.s.total - key0);
      wait_o();
#pragma unroll 1
      for (int c = C::kDims * half; c < C::kDims * (half + 1); c += 16) {
        uint32_t o[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = 0;
        if (!first) {
          tmem_ld16(row_tmem + C::kColO + c, o);
          ptx::tmem_wait_ld();
        }
#pragma unroll 1
        for (int k = 0; k < keys; ++k) {
          if (hidden >> k & 1) continue;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float y = v_in_memory<C>(v + (int64_t)k * C::kRowBytes, c + e);
            // the weight of a seen key is positive: it leaves y as it is
            if (!(fabsf(y) <= FLT_MAX)) o[e] = __float_as_uint(__uint_as_float(o[e]) + y);
          }
        }
        __syncwarp();
        ptx::tmem_st16(row_tmem + C::kColO + c, o);
      }
    }
  }
  ptx::tmem_wait_st();
}

template <class C>
__global__ void __launch_bounds__(C::kWideThreads, C::kCtas)
    tree_decode_wide_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw_smem[];
  __shared__ struct {
    // [i & 1] for unit i: a barrier's next phase waits for its last one's readers
    uint64_t kv_full[2], s_full[2], p_full[2], o_done[2], q_full, drain[2];
    uint32_t tmem;
    int odd[2];  // the last unit in this buffer whose V is not finite
    // read in pairs
    alignas(16) float k_scale[2][C::kKeys];
    alignas(16) float k_mid[2][C::kKeys];
    alignas(16) float v_scale[2][C::kKeys];
    alignas(16) float v_mid[2][C::kKeys];
    float v_top[2][2];  // the largest magnitude of a scale of V's rows 0-31 and 32-63
    float swap[2][C::kHalves == 2 ? C::kWeighers : 1];
  } sh;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  // until the host clears it; one answer for all, as warps wait for one another below
  if (__syncthreads_or(ptx::timeout_flagged(p.status))) return;
  if (tid == 0) p.split[blockIdx.x].b = -1;  // for the joining kernel

  int64_t begin, end, all;
  Cursor<C::kKeys> cur = share<C::kKeys>(p, begin, end, all);
  const int64_t units = end - begin;
  if (units <= 0) return;
  const uint32_t work = (ptx::smem_u32(raw_smem) + 1023) & ~1023u;
  const uint32_t q_at = work, kv_at = work + C::kSlabs * C::kQSlab;
  auto bar = [](uint64_t &b) { return ptx::smem_u32(&b); };
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar(sh.kv_full[i]), kLoaders);
      ptx::mbar_init(bar(sh.s_full[i]), 2);  // the products, and their issuer
      ptx::mbar_init(bar(sh.p_full[i]), C::kWeighers);
      ptx::mbar_init(bar(sh.o_done[i]), 1);
      ptx::mbar_init(bar(sh.drain[i]), 1);
      sh.odd[i] = -1;
    }
    ptx::mbar_init(bar(sh.q_full), C::kWeighers);
    ptx::fence_barrier_init();
  }
  if (warp == 0) {
    ptx::tmem_alloc(ptx::smem_u32(&sh.tmem), C::kCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = sh.tmem;
  constexpr int kRest = C::kWeighers / 32;  // the first warp that makes no weights

  if (warp >= kRest + 2) {
    // -------------------------------------------------------------- products
    // The warp waits in step; lane 0 issues.
    const uint32_t leader = (tid & 31) == 0;
    auto wait = [&](uint64_t &b, uint32_t parity) {
      return __all_sync(0xffffffffu, ptx::mbar_wait(bar(b), parity, p.status)) != 0;
    };
    bool ok = true;
    if (warp == kRest + 2) {
      const uint32_t idesc = idesc_wide(C::kBf16Rows, 64, false);
      uint32_t segment = 0;
#pragma unroll 1
      for (int64_t i = 0; i < units && ok; ++i) {
        const int buf = (int)(i & 1);
        const bool first = i == 0 || cur.u == 0;
        ok = wait(sh.kv_full[buf], (uint32_t)(i >> 1) & 1) &&
             (!first || wait(sh.q_full, segment & 1)) &&
             // S had P of the unit before last
             (i < 2 || wait(sh.o_done[buf], (uint32_t)((i - 2) >> 1) & 1));
        if (ok) {
          ptx::tc_fence_after();
          const uint32_t k = kv_at + buf * C::kBuf;
#pragma unroll
          for (int kk = 0; kk < C::D / 16; ++kk)
            mma_ss_warp(leader, tmem + C::kColS + 64 * buf,
                        ptx::smem_desc_sw128(q_at + kk / 4 * C::kQSlab + kk % 4 * 32, 16, 1024),
                        ptx::smem_desc_sw128(k + kk / 4 * C::kSlab + kk % 4 * 32, 16, 1024), idesc,
                        kk > 0);
          commit_warp(leader, bar(sh.s_full[buf]));
          // which has waited for the rows: so have, then, the weights' threads
          if (leader) ptx::mbar_arrive(bar(sh.s_full[buf]));
        }
        segment += first;
        cur.next(p);
      }
    } else {
      const uint32_t idesc = idesc_wide(C::kBf16Rows, C::D, true);
#pragma unroll 1
      for (int64_t i = 0; i < units && ok; ++i) {
        const int buf = (int)(i & 1);
        bool first = i == 0 || cur.u == 0;
        ok = wait(sh.kv_full[buf], (uint32_t)(i >> 1) & 1) &&
             wait(sh.p_full[buf], (uint32_t)(i >> 1) & 1);
        if (ok) {
          ptx::tc_fence_after();
          // the rows' threads have begun O themselves where V is odd
          first = first && sh.odd[buf] != (int)(i & 0x7fffffff);
          const uint32_t v = kv_at + buf * C::kBuf + C::kSlabs * C::kSlab;
#pragma unroll
          for (int term = C::kBf16Rows ? 1 : 0; term >= 0; --term)
#pragma unroll
            for (int kk = 0; kk < C::kKeys / 16; ++kk)  // 16 keys are two 8-row atoms
              mma_ts_warp(leader, tmem + C::kColO, tmem + C::kColS + 64 * buf + 32 * term + kk * 8,
                          ptx::smem_desc_sw128(v + kk * 2048, C::kSlab, 1024), idesc,
                          !first || kk > 0 || (C::kBf16Rows && term == 0));
          commit_warp(leader, bar(sh.o_done[buf]));
        }
        cur.next(p);
      }
    }
    if (!ok) {  // every product issued has to end before the memory goes
      commit_warp(leader, bar(sh.drain[warp - kRest - 2]));
      ptx::mbar_wait_drain(bar(sh.drain[warp - kRest - 2]), 0);
    }
  } else if (warp >= kRest) {
    // --------------------------------------------------------- rows of K and V
    const int t = tid - C::kWeighers;
    constexpr int kRowPieces = C::kRowBytes / 16;
    Cursor<C::kKeys> ahead = cur;
    uint4 held[C::kBf16Rows ? 1 : 2 * C::kPieces];  // codes of K, then of V
    uint32_t held_k = 0, held_v = 0;                // scales of row t
    // The unit fetched next, from this thread's first piece, which the others
    // follow kLoaders pieces apart.
    const int row0 = t / kRowPieces, col0 = t % kRowPieces;
    constexpr int kApart = kLoaders / kRowPieces;  // rows
    static_assert(kLoaders % kRowPieces == 0 && kApart >= 4, "pieces");
    // bytes from a piece of row row0 to the same of row row0 + j kApart; the
    // swizzle changes where rows are 4 apart
    auto to_piece = [&](uint32_t at, int j) {
      return (at ^ (j * kApart & 7) << 4) + j * kApart * 128;
    };
    const uint32_t to0 = kv_at + piece(row0, col0, C::kSlab);
    const uint8_t *k_at, *v_at, *ks_at = nullptr, *vs_at = nullptr;
    auto aim = [&]() {
      const int64_t row = ahead.b * p.c.sb + ahead.h * p.c.sh + (int64_t)ahead.u * C::kKeys;
      k_at = p.c.k + row * C::kRowBytes + t * 16;
      v_at = p.c.v + row * C::kRowBytes + t * 16;
      if constexpr (C::kScaled) {
        ks_at = p.c.k_scale + (row + t) * 4;
        vs_at = p.c.v_scale + (row + t) * 4;
      }
    };
    aim();
    // Its rows, to the buffer (bf16) or to be held.
    auto fetch = [&](int buf) {
      const int live = ahead.s.total - ahead.u * C::kKeys;
#pragma unroll
      for (int j = 0; j < C::kPieces; ++j) {
        const bool use = row0 + j * kApart < live;
        if constexpr (C::kBf16Rows) {
          const uint32_t to = to_piece(to0 + buf * C::kBuf, j);
          cp_async16(to, use ? k_at + j * 16 * kLoaders : p.c.k, use);
          cp_async16(to + C::kSlabs * C::kSlab, use ? v_at + j * 16 * kLoaders : p.c.v, use);
        } else {
          held[j] = held[C::kPieces + j] = make_uint4(0, 0, 0, 0);
          if (use) {
            held[j] = *reinterpret_cast<const uint4 *>(k_at + j * 16 * kLoaders);
            held[C::kPieces + j] = *reinterpret_cast<const uint4 *>(v_at + j * 16 * kLoaders);
          }
        }
      }
      if constexpr (C::kBf16Rows) {
        cp_async_commit();
        // the buffer after next is not free yet: its rows wait in L2
        constexpr int kUnit = C::kKeys * C::kRowBytes;
#pragma unroll
        for (int j = 0; j < C::kPieces; ++j)
          if (t % 8 == 0 && C::kKeys + row0 + j * kApart < live) {
            asm volatile("prefetch.global.L2 [%0];" ::"l"(k_at + kUnit + j * 16 * kLoaders));
            asm volatile("prefetch.global.L2 [%0];" ::"l"(v_at + kUnit + j * 16 * kLoaders));
          }
      } else {
        held_k = held_v = 0;
        if (t < live) {
          held_k = *reinterpret_cast<const uint32_t *>(ks_at);
          held_v = *reinterpret_cast<const uint32_t *>(vs_at);
        }
      }
      if (ahead.next(p)) {
        if (ahead.b < (int)p.c.B) aim();
      } else {
        k_at += C::kKeys * C::kRowBytes;
        v_at += C::kKeys * C::kRowBytes;
        if constexpr (C::kScaled) {
          ks_at += C::kKeys * 4;
          vs_at += C::kKeys * 4;
        }
      }
    };
    // Puts the rows held into buffer `buf` as f16.  tail: what is not finite in V
    // becomes 0; returns whether there was any.
    auto place_rows = [&](int buf, bool tail) -> bool {
      bool odd = false;
      if constexpr (C::kBf16Rows) {
        if (tail) {  // this thread's own pieces have arrived
#pragma unroll
          for (int j = 0; j < C::kPieces; ++j) {
            const uint32_t from = to_piece(to0 + buf * C::kBuf, j) + C::kSlabs * C::kSlab;
            const uint4 y = lds128(from);
            uint32_t w[4] = {y.x, y.y, y.z, y.w};
            bool here = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u, here = true;
              if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu, here = true;
            }
            if (here) sts128(from, make_uint4(w[0], w[1], w[2], w[3]));
            odd = odd || here;
          }
        }
      } else {
        constexpr int kParts = C::kFmt == WFATTN_CACHE_E4M3 ? 2 : 4;  // f16 pieces of one
        uint32_t part[kParts];
#pragma unroll
        for (int e = 0; e < kParts; ++e)
          part[e] = kv_at + buf * C::kBuf + piece(row0, kParts * col0 + e, C::kSlab);
#pragma unroll
        for (int j = 0; j < 2 * C::kPieces; ++j) {
          const uint32_t half = j < C::kPieces ? 0 : C::kSlabs * C::kSlab;
          const uint32_t w[4] = {held[j].x, held[j].y, held[j].z, held[j].w};
          if constexpr (C::kFmt == WFATTN_CACHE_E4M3) {
            uint32_t f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = ptx::e4m3x2_to_f16x2(w[e / 2] >> (16 * (e & 1)));
            if (tail && j >= C::kPieces) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                if ((f[e] & 0x7c00u) == 0x7c00u) f[e] &= 0xffff0000u, odd = true;
                if ((f[e] & 0x7c000000u) == 0x7c000000u) f[e] &= 0xffffu, odd = true;
              }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
              sts128(to_piece(part[e], j % C::kPieces) + half,
                     make_uint4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              sts128(to_piece(part[e], j % C::kPieces) + half,
                     make_uint4(int4_f16x2<false>(w[e]), int4_f16x2<true>(w[e]),
                                int4_f16x2<false>(w[e] >> 8), int4_f16x2<true>(w[e] >> 8)));
          }
        }
        // K's scale is NaN where it is not finite: a score of -inf would hide the key
        if constexpr (C::kFmt == WFATTN_CACHE_E4M3) {
          const float ks = __uint_as_float(held_k);
          sh.k_scale[buf][t] = ks + (ks - ks);
          sh.v_scale[buf][t] = __uint_as_float(held_v);
        } else {
          const float ks = ptx::bf16_lo(held_k), vs = ptx::bf16_lo(held_v);
          sh.k_scale[buf][t] = ks + (ks - ks);
          sh.v_scale[buf][t] = vs;
          sh.k_mid[buf][t] = fmaf(8.f, ks, ptx::bf16_hi(held_k));
          sh.v_mid[buf][t] = fmaf(8.f, vs, ptx::bf16_hi(held_v));
        }
        // the bits of magnitudes order like them; NaN does not count
        uint32_t top = (C::kFmt == WFATTN_CACHE_E4M3 ? held_v : held_v << 16) & 0x7fffffffu;
        top = __reduce_max_sync(0xffffffffu, top > 0x7f800000u ? 0u : top);
        if (t % 32 == 0) sh.v_top[buf][t / 32] = __uint_as_float(top);
      }
      return odd;
    };
    if constexpr (!C::kBf16Rows) fetch(0);
#pragma unroll 1
    for (int64_t i = 0; i < units; ++i) {
      const int buf = (int)(i & 1);
      // the buffer is free after P V of the unit before last
      if (i >= 2 &&
          !ptx::mbar_wait(bar(sh.o_done[buf]), (uint32_t)((i - 2) >> 1) & 1, p.status))
        break;
      if constexpr (C::kBf16Rows) {
        fetch(buf);
        cp_async_wait<0>();
      }
      if (place_rows(buf, (cur.u + 1) * C::kKeys > cur.s.len))
        sh.odd[buf] = (int)(i & 0x7fffffff);
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(bar(sh.kv_full[buf]));
      if (!C::kBf16Rows && i + 1 < units) fetch(0);
      cur.next(p);
    }
    if constexpr (C::kBf16Rows) cp_async_wait<0>();
  } else {
    // ---------------------------------------------------- weights, and results
    // Threads of a TMEM lane, 128 apart, have a row; each of two half of its keys and columns.
    const int row = tid % kThreads, half = tid / kThreads, quad = warp % 4;
    const uint32_t row_tmem = tmem + ((uint32_t)(quad * 32) << 16);
    int turn = 0;
    // Every pass through here is the same for both: it depends on no wait.
    auto swap = [&](float x) {
      turn ^= 1;
      return swap_halves(x, &sh.swap[turn][tid], &sh.swap[turn][tid ^ kThreads], 1 + quad);
    };
    bool headed = cur.u == 0, failed = false;
    auto wait = [&](uint64_t &b, uint32_t parity) {
      if (!failed && !ptx::mbar_wait(bar(b), parity, p.status)) failed = true;
    };
    int64_t i = 0;
#pragma unroll 1
    while (i < units) {  // a segment, or the part of it in this share
      // ---- the query row of this thread as an operand, scaled into f16's range
      const int r = cur.tile * C::kRows + row;
      const bool idle = cur.tile * C::kRows + quad * 32 >= p.R;  // both warps
      float qf = p.scale_log2, qsum = 0.f;
      uint64_t word = 0;
      {
        const int hg = over_T(p, r), node = r - hg * p.T;
        const uint16_t *q = reinterpret_cast<const uint16_t *>(p.q) + cur.b * p.qs.b +
                            ((int64_t)cur.h * p.G + hg) * p.qs.h + node * p.qs.s + C::kDims * half;
        uint32_t w[C::kDims / 2];
#pragma unroll
        for (int c = 0; c < C::kDims / 2; ++c) w[c] = 0;
        if (r < p.R) {
          word = p.tree ? p.tree[cur.b * p.tree_stride + node] : (2ull << node) - 1;
          if (p.q_vec) {
#pragma unroll
            for (int c = 0; c < C::kDims / 8; ++c) {
              const uint4 y = reinterpret_cast<const uint4 *>(q)[c];
              w[4 * c] = y.x, w[4 * c + 1] = y.y, w[4 * c + 2] = y.z, w[4 * c + 3] = y.w;
            }
          } else {
#pragma unroll
            for (int c = 0; c < C::kDims / 2; ++c) w[c] = q[2 * c] | (uint32_t)q[2 * c + 1] << 16;
          }
        }
        if constexpr (!C::kBf16Rows) {
          uint32_t top = 0;
#pragma unroll
          for (int c = 0; c < C::kDims / 2; ++c) top = __vmaxu2(top, w[c] & 0x7fff7fffu);
          top = max(top >> 16, top & 0xffffu) >> 7;  // exponent field
          int e = (int)top;
          if constexpr (C::kHalves == 2) e = max(e, __float_as_int(swap(__int_as_float(e))));
          const int f = min(max(268 - e, 1), 253);  // 2^14 <= top * mul < 2^15
          const float mul = __uint_as_float((uint32_t)f << 23);
          // not 0, as a hidden score of -inf times that is NaN
          qf = fmaxf(p.scale_log2 * __uint_as_float((uint32_t)(254 - f) << 23),
                     __uint_as_float(1));
#pragma unroll
          for (int c = 0; c < C::kDims / 8; ++c) {
            float x[8];
#pragma unroll
            for (int v = 0; v < 8; ++v) {
              const uint32_t y = w[4 * c + v / 2];
              const int at = C::kFmt == WFATTN_CACHE_INT4 ? int4_place(v) : v;
              x[at] = (v & 1 ? ptx::bf16_hi(y) : ptx::bf16_lo(y)) * mul;
              qsum += x[at];
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) w[4 * c + v] = pack_f16x2(x[2 * v], x[2 * v + 1]);
          }
          if constexpr (C::kHalves == 2) qsum += swap(qsum);
        }
#pragma unroll
        for (int c = 0; c < C::kDims / 8; ++c)
          sts128(q_at + piece(row, C::kDims / 8 * half + c, C::kQSlab),
                 make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(bar(sh.q_full));
      float m = -FLT_MAX, l = 0.f, om = 0.f;
      float vinv = __uint_as_float(253u << 23);  // as in Warp
      bool first = true, done;
#pragma unroll 1
      while (true) {  // a unit
        const int buf = (int)(i & 1);
        const uint32_t parity = (uint32_t)(i >> 1) & 1;
        wait(sh.s_full[buf], parity);
        ptx::tc_fence_after();
        const bool odd = sh.odd[buf] == (int)(i & 0x7fffffff);
        __syncwarp();
        // after a wait that failed as before it: the other half's warp counts on this one
        if (!idle) {
          const float vtop = C::kScaled ? fmaxf(sh.v_top[buf][0], sh.v_top[buf][1]) : 0.f;
          const int k0 = C::kMine * half;
          auto wait_o = [&]() {
            if (i > 0) wait(sh.o_done[buf ^ 1], (uint32_t)((i - 1) >> 1) & 1);
            ptx::tc_fence_after();
            __syncwarp();
          };
          if ((cur.u + 1) * C::kKeys > cur.s.len)
            weigh<C, true>(p, cur, half, row_tmem, row_tmem + C::kColS + 64 * buf,
                           cur.u * C::kKeys, odd, word, qf, qsum, sh.k_scale[buf] + k0,
                           sh.k_mid[buf] + k0, sh.v_scale[buf] + k0, sh.v_mid[buf] + k0, vtop,
                           first, m, l, om, vinv, swap, wait_o);
          else
            weigh<C, false>(p, cur, half, row_tmem, row_tmem + C::kColS + 64 * buf,
                            cur.u * C::kKeys, odd, word, qf, qsum, sh.k_scale[buf] + k0,
                            sh.k_mid[buf] + k0, sh.v_scale[buf] + k0, sh.v_mid[buf] + k0, vtop,
                            first, m, l, om, vinv, swap, wait_o);
        }
        ptx::tc_fence_before();
        ptx::mbar_arrive(bar(sh.p_full[buf]));
        first = false;
        done = cur.u + 1 == cur.s.units;
        if (done || i + 1 == units) break;
        ++i;
        ++cur.u;
      }

      // ---- the segment's end
      wait(sh.o_done[i & 1], (uint32_t)(i >> 1) & 1);
      ptx::tc_fence_after();
      const bool whole = done && headed;
      if constexpr (C::kHalves == 2) {
        l += swap(l);
        om += swap(om);
      }
      const int64_t slot = (int64_t)blockIdx.x * 2 + (headed ? 1 : 0);
      if (!idle && __all_sync(0xffffffffu, !failed)) {
        bool live = false;
        uint8_t *to = out_row(p, cur.b, cur.h, r, cur.s.n, 2, live);
        float *part = p.part + (slot * C::kRows + row) * C::D;
        const float back = C::kScaled ? 1.f / vinv : 1.f;
        const bool some = live && l != 0.f;
        const float inv = 1.f / l;
#pragma unroll 1
        for (int c = C::kDims * half; c < C::kDims * (half + 1); c += 32) {
          uint32_t o[32];
          ptx::tmem_ld32(row_tmem + C::kColO + c, o);
          ptx::tmem_wait_ld();
          float x[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int at = C::kFmt == WFATTN_CACHE_INT4 ? (e & ~7) + int4_place(e & 7) : e;
            x[e] = C::kScaled ? fmaf(__uint_as_float(o[at]), back, om) : __uint_as_float(o[at]);
          }
          if (to && whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              store_out4<false>(p, to, c + e,
                                some ? make_float4(x[e] * inv, x[e + 1] * inv, x[e + 2] * inv,
                                                   x[e + 3] * inv)
                                     : make_float4(0.f, 0.f, 0.f, 0.f));
          } else if (to) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4 *>(part + c + e) =
                  make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
          }
        }
        if (to && !whole && half == 0) {
          float *ml = p.part + (int64_t)p.ctas * 2 * C::kRows * C::D + (slot * C::kRows + row) * 2;
          ml[0] = m;
          ml[1] = l;
        }
      }
      ptx::tc_fence_before();  // O may be written again after this thread's next p_full
      if (!done && headed && tid == 0)
        p.split[blockIdx.x] = split_of(p, cur, begin + i - cur.u, all);
      headed = true;
      cur.next(p);
      ++i;
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, C::kCols);
  }
}

// ------------------------------------------------------------------ launch

template <class C>
cudaError_t launch_wide(Params p, void *workspace, const DeviceInfo &dev, cudaStream_t stream) {
  prepare<C>(p, workspace, dev);
  const cudaError_t err = ensure_smem_attr(
      reinterpret_cast<const void *>(tree_decode_wide_kernel<C>), C::kSmem, dev.device);
  if (err != cudaSuccess) return err;
  tree_decode_wide_kernel<C><<<p.ctas, C::kWideThreads, C::kSmem, stream>>>(p);
  return launch_join<C>(p, stream);
}

}  // namespace tree
}  // namespace wfattn
