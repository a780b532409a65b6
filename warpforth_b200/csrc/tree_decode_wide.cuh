// tree_decode_wide.cuh -- tree_decode for many query rows a cache head: the
// products on tcgen05 tensor cores.
//
// A CTA takes up to 128 query rows of one cache head (one TMEM lane, and one
// thread, a row) and walks its keys in blocks of 64:
//
//   S [128 x 64]   = Q [128 x D] K^T         both operands in shared memory
//   O [128 x D]   += P [128 x 64] V          P in tensor memory
//
// K and V lie in shared memory as 16-bit rows in the 128-byte swizzle that the
// operands have, K along a row and V across rows.  bf16 rows arrive there by
// cp.async; the codes of e4m3 and int4 rows come through registers, a block
// ahead, and are written as f16 (exactly; int4 as u - 8) while the products of
// the block before run.  Scales, weights, lazy maximum and the split of work
// are those of tree_decode.cuh; bf16 weights take two products (two terms).
//
// Per block and CTA: Q K^T; when S is there its weights, into tensor memory;
// P V, and meanwhile the next block's rows into the other buffer.  A thread's 64 exponentials
// (16 a clock and SM) bound it, so two CTAs an SM, each waiting for its own
// products, fill each other's gaps.  TMEM columns: S 64, P 32 (and 32 of second
// terms), O 64 or 128: 256 a CTA.
#pragma once

#include "tree_decode.cuh"

namespace wfattn {
namespace tree {

template <int kFmt_, int D_>
struct WideCfg {
  static constexpr int kFmt = kFmt_, D = D_, kRows = 128, kKeys = 64, kCtas = 2;
  static constexpr bool kF32 = false, kWide = true;
  static constexpr bool kBf16Rows = kFmt == WFATTN_CACHE_BF16;
  static constexpr bool kScaled = !kBf16Rows;
  static constexpr int kRowBytes = CacheRow<kFmt, D>::kBytes;
  static constexpr int kSlabs = D / 64;               // 128-byte wide slabs of an operand
  static constexpr int kSlab = kKeys * 128;           // bytes of a slab of K or V
  static constexpr int kQSlab = kRows * 128;
  static constexpr int kBuf = 2 * kSlabs * kSlab;     // K and V of a block
  static constexpr int kPieces = kKeys * (kBf16Rows ? 2 * D : kRowBytes) / 16 / kThreads;
  static constexpr int kWork = kSlabs * kQSlab + 2 * kBuf;
  static constexpr int kSmem = kWork + 1024;          // and room to align
  static constexpr uint32_t kColS = 0, kColP = 64, kColP2 = 96, kColO = 128, kCols = 256;
  static_assert(kSmem <= 227 * 1024 / kCtas - 3072, "two CTAs an SM");
};

__device__ __forceinline__ uint32_t idesc_wide(bool bf16, bool b_mn) {
  // M 128, N 64, f32 accumulation; formats f16 (0) or bf16 (1)
  return ptx::idesc_bf16_f32(128, 64, 0, b_mn ? 1 : 0) & (bf16 ? ~0u : ~((1u << 7) | (1u << 10)));
}

// Byte offset of the 16-byte piece c (8 values) of row r in an operand whose
// slabs have `slab` bytes.
__device__ __forceinline__ uint32_t piece(int r, int c, int slab) {
  return (c >> 3) * slab + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// int4 rows are unpacked as pairs of codes n, n + 4 of a word: value `v` of a
// row's eight is at place `i`.
__device__ __forceinline__ constexpr int int4_place(int v) { return 2 * (v & 3) + (v >> 2); }

__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

// A value of V in memory, unscaled; used where a row is not finite.
template <class C>
__device__ __forceinline__ float v_in_memory(const uint8_t *row, int d) {
  if constexpr (C::kBf16Rows) return ptx::bf16_lo(reinterpret_cast<const uint16_t *>(row)[d]);
  return ptx::f16x2_to_f32(ptx::e4m3x2_to_f16x2(row[d])).x;
}

__device__ __forceinline__ void tmem_load64(uint32_t at, uint32_t (&s)[64]) {
  ptx::tmem_ld_32x32b_x64(at, s);
  ptx::tmem_wait_ld();
}

// A thread's row of S to weights in tensor memory: maximum, sum and (int4) the
// sum of weights times minima go on in m, l and om.
template <class C>
__device__ __forceinline__ void weigh(const Params &p, const Cursor<C::kKeys> &cur,
                                      uint32_t (&s)[64], uint32_t row_tmem, int key0, bool tail,
                                      bool odd, uint64_t word, float qf, float qsum,
                                      const float *k_scale, const float *k_mid,
                                      const float *v_scale, const float *v_mid, bool first,
                                      float &m, float &l, float &om, float &vinv) {
  const int lane = threadIdx.x & 31;
  // scores before qf, which is positive
  const uint64_t qsum2 = ptx::f2_pack(qsum, qsum);
  if constexpr (C::kScaled) {
#pragma unroll
    for (int k = 0; k < 64; k += 2) {
      const uint64_t ks = *reinterpret_cast<const uint64_t *>(k_scale + k);
      const uint64_t x = ptx::f2_pack(__uint_as_float(s[k]), __uint_as_float(s[k + 1]));
      uint64_t y;
      if constexpr (C::kFmt == WFATTN_CACHE_INT4)
        y = ptx::f2_fma(x, ks, ptx::f2_mul(*reinterpret_cast<const uint64_t *>(k_mid + k), qsum2));
      else
        y = ptx::f2_mul(x, ks);
      float a, b;
      ptx::f2_unpack(y, a, b);
      s[k] = __float_as_uint(a);
      s[k + 1] = __float_as_uint(b);
    }
  }
  if (tail) {
    const int node0 = key0 - cur.s.len;
#pragma unroll
    for (int k = 0; k < 64; ++k) {
      const int node = node0 + k;
      if (node >= 0 && (node >= cur.s.n || !(word >> node & 1))) s[k] = 0xff800000u;
    }
  }
  float high = -INFINITY;
#pragma unroll
  for (int k = 0; k < 64; k += 2)
    high = ptx::fmax3(high, __uint_as_float(s[k]), __uint_as_float(s[k + 1]));
  float vtop = 0.f;
  if constexpr (C::kScaled) {
    vtop = fmaxf(v_scale[lane], v_scale[lane + 32]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, x));
  }
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
#pragma unroll 1
      for (int c = 0; c < C::D; c += 32) {
        uint32_t o[32];
        ptx::tmem_ld32(row_tmem + C::kColO + c, o);
        ptx::tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e)
          o[e] = __float_as_uint(__uint_as_float(o[e]) * (f * ratio));
        ptx::tmem_st32(row_tmem + C::kColO + c, o);
      }
    }
  }
  const uint64_t qf2 = ptx::f2_pack(qf, qf), m2 = ptx::f2_pack(-m, -m);
  const uint64_t vinv2 = ptx::f2_pack(vinv, vinv);
  uint64_t l2 = ptx::f2_pack(0.f, 0.f), om2 = l2;
  uint32_t hi[32];
#pragma unroll
  for (int k = 0; k < 64; k += 2) {
    const uint64_t d =
        ptx::f2_fma(ptx::f2_pack(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), qf2, m2);
    float a, b;
    ptx::f2_unpack(d, a, b);
    a = ptx::ex2_approx(a);
    b = ptx::ex2_approx(b);
    const uint64_t w = ptx::f2_pack(a, b);
    l2 = ptx::f2_add(l2, w);
    if constexpr (C::kScaled) {
      const bool hide_a = tail && s[k] == 0xff800000u, hide_b = tail && s[k + 1] == 0xff800000u;
      if constexpr (C::kFmt == WFATTN_CACHE_INT4) {
        uint64_t mid = *reinterpret_cast<const uint64_t *>(v_mid + k);
        if (tail) {  // a scale may be NaN
          float x, y;
          ptx::f2_unpack(mid, x, y);
          mid = ptx::f2_pack(hide_a ? 0.f : x, hide_b ? 0.f : y);
        }
        om2 = ptx::f2_fma(w, mid, om2);
      }
      ptx::f2_unpack(
          ptx::f2_mul(w, ptx::f2_mul(*reinterpret_cast<const uint64_t *>(v_scale + k), vinv2)), a,
          b);
      if (hide_a) a = 0.f;
      if (hide_b) b = 0.f;
      hi[k / 2] = pack_f16x2(a, b);
    } else {
      hi[k / 2] = ptx::pack_bf16x2(a, b);
      s[k / 2] = ptx::pack_bf16x2(a - ptx::bf16_lo(hi[k / 2]), b - ptx::bf16_hi(hi[k / 2]));
    }
  }
  float a, b;
  ptx::f2_unpack(l2, a, b);
  l += a + b;
  if constexpr (C::kFmt == WFATTN_CACHE_INT4) {
    ptx::f2_unpack(om2, a, b);
    om += a + b;
  }
  ptx::tmem_st32(row_tmem + C::kColP, hi);
  if constexpr (C::kBf16Rows) {
    uint32_t lo[32];
#pragma unroll
    for (int k = 0; k < 32; ++k) lo[k] = s[k];
    ptx::tmem_st32(row_tmem + C::kColP2, lo);
  }
  if constexpr (C::kFmt != WFATTN_CACHE_INT4) {
    if (odd) {
      // What is not finite in V was put to zero in the operand, where a weight
      // of 0 would spread it: rows that see its key get it here.
      const uint8_t *v =
          p.c.v + (cur.b * p.c.sb + cur.h * p.c.sh + (int64_t)key0) * C::kRowBytes;
      const int keys = min(64, cur.s.total - key0);
#pragma unroll 1
      for (int c = 0; c < C::D; c += 32) {
        uint32_t o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0;
        if (!first) {
          ptx::tmem_ld32(row_tmem + C::kColO + c, o);
          ptx::tmem_wait_ld();
        }
#pragma unroll 1
        for (int k = 0; k < keys; ++k) {
          const int node = key0 + k - cur.s.len;
          if (node >= 0 && (node >= cur.s.n || !(word >> node & 1))) continue;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float y = v_in_memory<C>(v + (int64_t)k * C::kRowBytes, c + e);
            // a weight that is seen is not negative, so what it gives is y, or
            // NaN where the weight may be 0 or the sums meet
            if (!(fabsf(y) <= FLT_MAX)) o[e] = __float_as_uint(__uint_as_float(o[e]) + y);
          }
        }
        ptx::tmem_st32(row_tmem + C::kColO + c, o);
      }
    }
  }
  ptx::tmem_wait_st();
}

template <class C>
__global__ void __launch_bounds__(kThreads, C::kCtas) 
    tree_decode_wide_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw_smem[];
  __shared__ uint64_t bar_s, bar_o, bar_drain;
  __shared__ uint32_t tmem_base;
  __shared__ __align__(16) float k_scale[2][C::kKeys], k_mid[2][C::kKeys];
  __shared__ __align__(16) float v_scale[2][C::kKeys], v_mid[2][C::kKeys];
  const int tid = threadIdx.x, warp = tid >> 5;
  if (ptx::timeout_flagged(p.status)) return;  // until the host clears it

  int64_t begin, end, all;
  Cursor<C::kKeys> cur = share<C::kKeys>(p, begin, end, all), ahead = cur;
  const int64_t units = end - begin;
  if (units <= 0) return;
  const uint32_t work = (ptx::smem_u32(raw_smem) + 1023) & ~1023u;
  uint8_t *room = raw_smem + (work - ptx::smem_u32(raw_smem));
  const uint32_t q_at = work, kv_at = work + C::kSlabs * C::kQSlab;
  if (tid == 0) {
    ptx::mbar_init(ptx::smem_u32(&bar_s), 1);
    ptx::mbar_init(ptx::smem_u32(&bar_o), 1);
    ptx::mbar_init(ptx::smem_u32(&bar_drain), 1);
    ptx::fence_barrier_init();
  }
  if (warp == 0) {
    ptx::tmem_alloc(ptx::smem_u32(&tmem_base), C::kCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tmem_base;
  const uint32_t row_tmem = tmem + ((uint32_t)(warp * 32) << 16);  // this thread's lane

  // ---- rows of K and V: the next unit's on their way
  uint4 held[C::kBf16Rows ? 1 : 2 * C::kPieces];  // codes of K, then of V
  uint32_t held_scale = 0;                        // threads 0-63: of K's rows, 64-127: V's
  int64_t to_fetch = units;
  auto fetch = [&](int buf) {
    if (to_fetch > 0) {
      --to_fetch;
      const int live = ahead.s.total - ahead.u * C::kKeys;
      const int64_t row =
          ahead.b * p.c.sb + ahead.h * p.c.sh + (int64_t)ahead.u * C::kKeys;
      const uint8_t *k = p.c.k + row * C::kRowBytes, *v = p.c.v + row * C::kRowBytes;
      constexpr int kRowPieces = C::kRowBytes / 16;
#pragma unroll
      for (int j = 0; j < C::kPieces; ++j) {
        const int i = tid + j * kThreads, r = i / kRowPieces, c = i % kRowPieces;
        const bool use = r < live;
        if constexpr (C::kBf16Rows) {
          const uint32_t to = kv_at + buf * C::kBuf + piece(r, c, C::kSlab);
          cp_async16(to, use ? k + i * 16 : p.c.k, use);
          cp_async16(to + C::kSlabs * C::kSlab, use ? v + i * 16 : p.c.v, use);
        } else {
          held[j] = held[C::kPieces + j] = make_uint4(0, 0, 0, 0);
          if (use) {
            held[j] = *reinterpret_cast<const uint4 *>(k + i * 16);
            held[C::kPieces + j] = *reinterpret_cast<const uint4 *>(v + i * 16);
          }
        }
      }
      if constexpr (C::kScaled) {
        const int r = tid % C::kKeys;
        const uint8_t *s = tid < C::kKeys ? p.c.k_scale : p.c.v_scale;
        held_scale = 0;
        if (r < live) held_scale = *reinterpret_cast<const uint32_t *>(s + (row + r) * 4);
      }
      ahead.next(p);
    }
    if constexpr (C::kBf16Rows) cp_async_commit();
  };
  // Puts the codes held into buffer `buf` as f16.  tail: what is not finite in V
  // becomes 0; returns whether there was any.
  auto place_rows = [&](int buf, bool tail) -> bool {
    bool odd = false;
    const uint32_t at = kv_at + buf * C::kBuf;
    if constexpr (C::kBf16Rows) {
      if (tail) {  // this thread's own pieces have arrived
#pragma unroll
        for (int j = 0; j < C::kPieces; ++j) {
          const int i = tid + j * kThreads;
          const uint32_t from = at + C::kSlabs * C::kSlab +
                                piece(i / (C::D / 8), i % (C::D / 8), C::kSlab);
          uint4 y = lds128(from);
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
      constexpr int kRowPieces = C::kRowBytes / 16;
#pragma unroll
      for (int j = 0; j < 2 * C::kPieces; ++j) {
        const int i = tid + j % C::kPieces * kThreads, r = i / kRowPieces, c = i % kRowPieces;
        const uint32_t base = at + (j < C::kPieces ? 0 : C::kSlabs * C::kSlab);
        const uint32_t w[4] = {held[j].x, held[j].y, held[j].z, held[j].w};
        if constexpr (C::kFmt == WFATTN_CACHE_E4M3) {
          uint32_t f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            f[e] = ptx::e4m3x2_to_f16x2(w[e / 2] >> (16 * (e & 1)));
          if (tail && j >= C::kPieces) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if ((f[e] & 0x7c00u) == 0x7c00u) f[e] &= 0xffff0000u, odd = true;
              if ((f[e] & 0x7c000000u) == 0x7c000000u) f[e] &= 0xffffu, odd = true;
            }
          }
          sts128(base + piece(r, 2 * c, C::kSlab), make_uint4(f[0], f[1], f[2], f[3]));
          sts128(base + piece(r, 2 * c + 1, C::kSlab), make_uint4(f[4], f[5], f[6], f[7]));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sts128(base + piece(r, 4 * c + e, C::kSlab),
                   make_uint4(int4_f16x2<false>(w[e]), int4_f16x2<true>(w[e]),
                              int4_f16x2<false>(w[e] >> 8), int4_f16x2<true>(w[e] >> 8)));
        }
      }
      const int r = tid % C::kKeys;
      float *s = tid < C::kKeys ? k_scale[buf] : v_scale[buf];
      float *m = tid < C::kKeys ? k_mid[buf] : v_mid[buf];
      if constexpr (C::kFmt == WFATTN_CACHE_E4M3) {
        s[r] = __uint_as_float(held_scale);
      } else {
        s[r] = ptx::bf16_lo(held_scale);
        m[r] = fmaf(8.f, ptx::bf16_lo(held_scale), ptx::bf16_hi(held_scale));
      }
    }
    return odd;
  };

  const uint32_t idesc_qk = idesc_wide(C::kBf16Rows, false);
  const uint32_t idesc_pv = idesc_wide(C::kBf16Rows, true);
  auto issue_qk = [&](int buf) {
    ptx::tc_fence_after();
#pragma unroll
    for (int kk = 0; kk < C::D / 16; ++kk)
      ptx::mma_ss(tmem + C::kColS,
                  ptx::smem_desc_sw128(q_at + kk / 4 * C::kQSlab + kk % 4 * 32, 16, 1024),
                  ptx::smem_desc_sw128(kv_at + buf * C::kBuf + kk / 4 * C::kSlab + kk % 4 * 32,
                                       16, 1024),
                  idesc_qk, kk > 0);
    ptx::tc_commit(ptx::smem_u32(&bar_s));
  };
  auto issue_pv = [&](int buf, bool first) {
    ptx::tc_fence_after();
    const uint32_t v = kv_at + buf * C::kBuf + C::kSlabs * C::kSlab;
#pragma unroll
    for (int term = C::kBf16Rows ? 1 : 0; term >= 0; --term)
#pragma unroll
      for (int kk = 0; kk < C::kKeys / 16; ++kk)
#pragma unroll
        for (int s = 0; s < C::kSlabs; ++s)
          ptx::mma_ts(tmem + C::kColO + 64 * s,
                      tmem + (term ? C::kColP2 : C::kColP) + kk * 8,
                      ptx::smem_desc_sw128(v + s * C::kSlab + kk * 2048, C::kSlab, 1024), idesc_pv,
                      !first || kk > 0 || (C::kBf16Rows && term == 0));
    ptx::tc_commit(ptx::smem_u32(&bar_o));
  };

  uint32_t phase_s = 0, phase_o = 0;  // of the next completion to wait for
  bool failed = false, pending = false;  // pending: a P V that was not waited for
  auto wait_o = [&]() {
    if (pending) {
      if (!ptx::mbar_wait(ptx::smem_u32(&bar_o), phase_o, p.status)) failed = true;
      phase_o ^= 1;
      pending = false;
      ptx::tc_fence_after();
    }
  };
  auto has_tail = [&](const Cursor<C::kKeys> &c) { return (c.u + 1) * C::kKeys > c.s.len; };

  // ---- the first unit
  fetch(0);
  if constexpr (C::kBf16Rows) cp_async_wait<0>();
  bool odd = place_rows(0, has_tail(cur));
  if constexpr (!C::kBf16Rows) fetch(0);
  int buf = 0;
  bool headed = cur.u == 0;
  int64_t i = 0;
#pragma unroll 1
  while (i < units && !failed) {  // a segment, or the part of it in this share
    // ---- the query row of this thread as an operand, scaled into f16's range
    const int r = cur.tile * C::kRows + tid;
    const bool idle = cur.tile * C::kRows + warp * 32 >= p.R;  // the whole warp
    float qf = p.scale_log2, qsum = 0.f;
    uint64_t word = 0;
    {
      const int hg = over_T(p, r), node = r - hg * p.T;
      const uint16_t *q = reinterpret_cast<const uint16_t *>(p.q) + cur.b * p.qs.b +
                          ((int64_t)cur.h * p.G + hg) * p.qs.h + node * p.qs.s;
      uint32_t w[C::D / 2];
#pragma unroll
      for (int c = 0; c < C::D / 2; ++c) w[c] = 0;
      if (r < p.R) {
        word = p.tree ? p.tree[cur.b * p.tree_stride + node] : (2ull << node) - 1;
        if (p.q_vec) {
#pragma unroll
          for (int c = 0; c < C::D / 8; ++c) {
            const uint4 y = reinterpret_cast<const uint4 *>(q)[c];
            w[4 * c] = y.x, w[4 * c + 1] = y.y, w[4 * c + 2] = y.z, w[4 * c + 3] = y.w;
          }
        } else {
#pragma unroll
          for (int c = 0; c < C::D / 2; ++c) w[c] = q[2 * c] | (uint32_t)q[2 * c + 1] << 16;
        }
      }
      if constexpr (!C::kBf16Rows) {
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < C::D / 2; ++c) top = __vmaxu2(top, w[c] & 0x7fff7fffu);
        const int e = (int)(max(top >> 16, top & 0xffffu) >> 7);  // exponent field
        const int f = min(max(268 - e, 1), 253);                  // 2^14 <= top * mul < 2^15
        const float mul = __uint_as_float((uint32_t)f << 23);
        qf = p.scale_log2 * __uint_as_float((uint32_t)(254 - f) << 23);
#pragma unroll
        for (int c = 0; c < C::D / 8; ++c) {
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
      }
#pragma unroll
      for (int c = 0; c < C::D / 8; ++c)
        sts128(q_at + piece(tid, c, C::kQSlab),
               make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
    }
    float m = -FLT_MAX, l = 0.f, om = 0.f;
    float vinv = __uint_as_float(253u << 23);  // as in Warp
    bool first = true, done;
#pragma unroll 1
    while (true) {  // a unit; its rows are in buffer `buf`
      ptx::fence_proxy_async_smem();
      ptx::tc_fence_before();
      odd = __syncthreads_or(odd);
      if (tid == 0) issue_qk(buf);
      wait_o();  // the other buffer, P and O are free
      if constexpr (C::kBf16Rows) fetch(buf ^ 1);
      if (!ptx::mbar_wait(ptx::smem_u32(&bar_s), phase_s, p.status)) failed = true;
      phase_s ^= 1;
      ptx::tc_fence_after();
      const int key0 = cur.u * C::kKeys;
      // waits end the same way in a warp's threads, or the CTA gives up below
      const bool work_here = !idle && __all_sync(0xffffffffu, !failed);
      if (work_here) {
        uint32_t s[64];
        tmem_load64(row_tmem + C::kColS, s);
        weigh<C>(p, cur, s, row_tmem, key0, has_tail(cur), odd != 0, word, qf, qsum, k_scale[buf],
                 k_mid[buf], v_scale[buf], v_mid[buf], first, m, l, om, vinv);
      }
      first = first && !odd;
      ptx::tc_fence_before();
      failed = __syncthreads_or(failed);
      if (failed) break;
      if (tid == 0) issue_pv(buf, first);
      pending = true;
      first = false;
      // ---- the next unit's rows, of this segment or the next one's
      done = cur.u + 1 == cur.s.units;
      Cursor<C::kKeys> next = cur;
      next.next(p);
      odd = false;
      if (i + 1 < units) {
        if constexpr (C::kBf16Rows) cp_async_wait<0>();
        odd = place_rows(buf ^ 1, has_tail(next));
        if constexpr (!C::kBf16Rows) fetch(0);
        buf ^= 1;
      }
      if (done || i + 1 == units) break;
      ++i;
      cur = next;
    }
    if (failed) break;

    // ---- the segment's end
    wait_o();
    failed = __syncthreads_or(failed);
    if (failed) break;
    const bool whole = done && headed;
    const int64_t slot = (int64_t)blockIdx.x * 2 + (headed ? 1 : 0);
    if (!idle) {
      bool live = false;
      uint8_t *to = out_row(p, cur.b, cur.h, r, cur.s.n, 2, live);
      float *part = p.part + (slot * C::kRows + tid) * C::D;
      const float back = C::kScaled ? 1.f / vinv : 1.f;
      const bool some = live && l != 0.f;
      const float inv = 1.f / l;
#pragma unroll 1
      for (int c = 0; c < C::D; c += 32) {
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
      if (to && !whole) {
        float *ml = p.part + (int64_t)p.ctas * 2 * C::kRows * C::D + (slot * C::kRows + tid) * 2;
        ml[0] = m;
        ml[1] = l;
      }
    }
    ptx::tc_fence_before();
    if (!whole) {  // as in tree_decode_kernel
      const int64_t s0 = begin + i - cur.u;
      const int first_cta = headed ? (int)blockIdx.x : (int)(((s0 + 1) * p.ctas - 1) / all);
      const int last_cta = (int)(((s0 + cur.s.units) * p.ctas - 1) / all);
      join<C>(p, cur.b, cur.h, cur.tile, cur.s.n, first_cta, last_cta,
              min(last_cta - first_cta + 1, cur.s.units), all, room);
    }
    __syncthreads();  // before the next segment's queries take the room, and O its sums
    headed = true;
    cur.next(p);
    ++i;
  }

  if constexpr (C::kBf16Rows) cp_async_wait<0>();
  if (failed && tid == 0) {  // every product issued has to end before the memory goes
    ptx::tc_commit(ptx::smem_u32(&bar_drain));
    ptx::mbar_wait_drain(ptx::smem_u32(&bar_drain), 0);
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
  tree_decode_wide_kernel<C><<<p.ctas, kThreads, C::kSmem, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace tree
}  // namespace wfattn
