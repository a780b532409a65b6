// cache_sm100.cu -- writing, reading and keeping rows of a key/value cache
// (formats: include/wfattn.h).
//
// All three are moves of rows, bound by HBM.  A row of D values is D/8 lanes'
// work, 8 values (16 or 32 bytes) a lane, so loads and stores are 4 to 32 bytes
// a lane and a warp touches whole 128-byte lines.  A row's largest magnitude
// (e4m3) or its extremes (int4) are shuffles over its lanes; nothing goes
// through shared memory.  Reading 983,040 e4m3 rows of 64 values of K and of V as
// bf16, with the zeros behind ragged lengths: 85 us, 6.3 TB/s; writing 429,000
// rows of 128 values (8 ragged prompts, 16 heads, K and V) from bf16: bf16 rows 70
// us and e4m3 66, at the rate of a copy, 4 bits 107, bound by issue slots.
#include "cache_format.cuh"

namespace wfattn {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsAtOnce = 4;  // of a lane group, in flight together

struct RowsParams {
  CacheView c;
  uint8_t *x[2];          // rows of new (or read) keys, values
  Strides3 xs[2];         // element strides
  uint32_t n, rows;       // rows a head, rows in all
  uint32_t tiles;         // blocks a head (long form)
  const int32_t *starts, *counts;
  bool zero_rest;
  unsigned int *status;
};

// Eight values of the caller's rows, as they are in memory.
template <bool kF32>
struct Raw {
  uint32_t w[kF32 ? 8 : 4];
};

// kVec: 16-byte aligned.
template <bool kF32, bool kVec>
__device__ __forceinline__ Raw<kF32> load_raw(const uint8_t *x) {
  Raw<kF32> r;
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < (kF32 ? 2 : 1); ++i) {
      const uint4 v = reinterpret_cast<const uint4 *>(x)[i];
      r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
    }
  } else if constexpr (kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = reinterpret_cast<const uint32_t *>(x)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r.w[i] = reinterpret_cast<const uint16_t *>(x)[2 * i] |
               (uint32_t)reinterpret_cast<const uint16_t *>(x)[2 * i + 1] << 16;
  }
  return r;
}

template <bool kF32>
__device__ __forceinline__ void to_f32(const Raw<kF32> &r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (kF32)
      f[i] = __uint_as_float(r.w[i]);
    else
      f[i] = i & 1 ? ptx::bf16_hi(r.w[i / 2]) : ptx::bf16_lo(r.w[i / 2]);
  }
}

template <bool kF32, bool kVec>
__device__ __forceinline__ void rows_store8(uint8_t *x, const float (&f)[8]) {
  if constexpr (kF32 && kVec) {
    *reinterpret_cast<float4 *>(x) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4 *>(x + 16) = make_float4(f[4], f[5], f[6], f[7]);
  } else if constexpr (kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<float *>(x)[i] = f[i];
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = ptx::pack_bf16x2(f[2 * i], f[2 * i + 1]);
    if constexpr (kVec) {
      *reinterpret_cast<uint4 *>(x) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        reinterpret_cast<uint16_t *>(x)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
    }
  }
}

// ---- extremes of a row; NaN wins both ways

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t min_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <bool kF32, int kLanes>
__device__ __forceinline__ void row_extremes(const Raw<kF32> &x, float &lo, float &hi) {
  if constexpr (kF32) {
    lo = hi = __uint_as_float(x.w[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      lo = min_nan(lo, __uint_as_float(x.w[i]));
      hi = max_nan(hi, __uint_as_float(x.w[i]));
    }
#pragma unroll
    for (int m = 1; m < kLanes; m <<= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, m));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    }
  } else {
    uint32_t l = x.w[0], h = x.w[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) l = min_nan_bf16x2(l, x.w[i]), h = max_nan_bf16x2(h, x.w[i]);
#pragma unroll
    for (int m = 1; m < kLanes; m <<= 1) {
      l = min_nan_bf16x2(l, __shfl_xor_sync(0xffffffffu, l, m));
      h = max_nan_bf16x2(h, __shfl_xor_sync(0xffffffffu, h, m));
    }
    lo = min_nan(ptx::bf16_lo(l), ptx::bf16_hi(l));
    hi = max_nan(ptx::bf16_lo(h), ptx::bf16_hi(h));
  }
}

// The largest magnitude of a row as f32 bits, which order like |x|: infinities
// and NaN are the largest.
template <bool kF32, int kLanes>
__device__ __forceinline__ uint32_t row_top(const Raw<kF32> &x) {
  uint32_t top = 0;
  if constexpr (kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, x.w[i] & 0x7fffffffu);
#pragma unroll
    for (int m = 1; m < kLanes; m <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
    return top;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __vmaxu2(top, x.w[i] & 0x7fff7fffu);
#pragma unroll
    for (int m = 1; m < kLanes; m <<= 1)
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, m));
    return max(top << 16, top & 0xffff0000u);
  }
}

// x as the nearest bf16 not above (kDown) or not below it; x finite.
template <bool kDown>
__device__ __forceinline__ float to_bf16_directed(float x) {
  const uint32_t cut = __float_as_uint(x) & 0xffff0000u;  // towards zero
  const float t = __uint_as_float(cut);
  const bool step = kDown ? t > x : t < x;
  return step ? __uint_as_float(cut + 0x10000u) : t;  // away from zero
}

// Stores 8 values of a row in the cache's format; the row's kLanes lanes call
// it together (every lane of the warp does, `live` or not).
template <int kFmt, bool kF32, int kLanes>
__device__ __forceinline__ void cache_store8(uint8_t *codes, uint8_t *scale, bool first, bool live,
                                             const Raw<kF32> &x) {
  float f[8];
  to_f32<kF32>(x, f);
  if constexpr (kFmt == WFATTN_CACHE_F32) {
    if (live) rows_store8<true, true>(codes, f);
  } else if constexpr (kFmt == WFATTN_CACHE_BF16) {
    if (live) rows_store8<false, true>(codes, f);
  } else if constexpr (kFmt == WFATTN_CACHE_E4M3) {
    const uint32_t top = row_top<kF32, kLanes>(x);
    const bool bad = top >= 0x7f800000u;
    // 448 = 1.75 * 2^8: the exponent of the smallest 2^e with |x| <= 448 2^e
    const int e = max((int)(top >> 23) - 135 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // x 2^-e is exact: one rounding
      w[i] = ptx::pack_e4m3x2(f[2 * i] * inv, f[2 * i + 1] * inv);
    if (!live) return;
    *reinterpret_cast<uint2 *>(codes) =
        bad ? make_uint2(0, 0) : make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    if (first)
      *reinterpret_cast<uint32_t *>(scale) = bad ? 0x7fc00000u : (uint32_t)(127 + e) << 23;
  } else {
    float lo, hi;
    row_extremes<kF32, kLanes>(x, lo, hi);
    const float m = to_bf16_directed<true>(lo);
    const float s = to_bf16_directed<false>(__fdiv_rn(__fsub_rn(hi, m), 15.f));
    // the largest bf16; a NaN or an infinity among the values, or a span past f32
    const bool bad = !(s <= 3.38953139e38f);
    // u = rint(fl(a / s)), a = fl(x - m) >= 0.  a <= 15 s (1 + 2^-23), so u is in
    // 0..15 without a clamp.  t = a (1 / s) + 1.5 2^23 holds a whole number r next
    // to a / s in its low bits, and e = a - r s is exact (r s has 12 bits) where
    // it matters: r is u while |e| stays below s / 2 by more than a quotient's
    // rounding; |e| = s / 2 is a tie, which a and s of few bits meet often, and
    // its quotient is exact; only else the division itself is needed.
    constexpr float kMagic = 12582912.f;
    const float inv = __frcp_rn(s), half = 0.5f * s, sure = half * (1.f - 0x1p-18f);
    const uint64_t m2 = ptx::f2_pack(-m, -m), magic2 = ptx::f2_pack(kMagic, kMagic);
    const uint64_t inv2 = ptx::f2_pack(inv, inv), less2 = ptx::f2_pack(-kMagic, -kMagic);
    const uint64_t s2 = ptx::f2_pack(-s, -s);
    float t[8], e[8], far = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint64_t a = ptx::f2_add(ptx::f2_pack(f[i], f[i + 1]), m2);
      const uint64_t y = ptx::f2_fma(a, inv2, magic2);
      ptx::f2_unpack(y, t[i], t[i + 1]);
      ptx::f2_unpack(ptx::f2_fma(ptx::f2_add(y, less2), s2, a), e[i], e[i + 1]);
      far = ptx::fmax3(far, fabsf(e[i]), fabsf(e[i + 1]));
    }
    if (!(far < sure) || !(inv < 1e38f)) {  // or 1 / s overflows, or s is 0
      bool divide = !(inv < 1e38f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = fabsf(e[i]);
        if (d == half)  // to the even neighbour
          t[i] += __float_as_uint(t[i]) & 1 ? copysignf(1.f, e[i]) : 0.f;
        else
          divide = divide || !(d < sure);
      }
      if (divide) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          t[i] = kMagic + (s > 0.f ? rintf(__fdiv_rn(__fsub_rn(f[i], m), s)) : 0.f);
      }
    }
    uint32_t w = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i) w = w * 16 + __float_as_uint(t[i]);
    w -= 0x4b400000u * 0x11111111u;  // the bits of kMagic in all of them
    if (!live) return;
    *reinterpret_cast<uint32_t *>(codes) = bad ? 0u : w;
    if (first)
      *reinterpret_cast<uint32_t *>(scale) =
          bad ? 0x7fc07fc0u : (__float_as_uint(s) >> 16) | (__float_as_uint(m) & 0xffff0000u);
  }
}

// Which of a head's rows i < n are live, and its first row's position: those in
// [from, to), at positions start + i.
struct Span {
  int64_t start;
  int from, to;
};
__device__ __forceinline__ Span live_rows(const RowsParams &p, uint32_t b, bool report) {
  const int n = (int)p.n, start = p.starts[b];
  const int count = p.counts ? p.counts[b] : n;
  Span s;
  s.start = start;
  s.to = min(max(count, 0), n);
  s.from = start < 0 ? (int)imin64(s.to, -(int64_t)start) : 0;
  const int last = (int)imax64(s.from, imin64(s.to, p.c.L - start));
  if (report && (count < 0 || count > n || (s.to > 0 && (start < 0 || last < s.to))))
    atomicOr(p.status, kDevBadRowMask);
  s.to = last;
  return s;
}

// Rows of K (or V) of one head: kLong, a block's share of them, contiguous, a
// lane group taking every kGroups-th; else one row a group, whichever head's.
template <int kFmt, int D, bool kF32, bool kVec, bool kWrite, bool kLong>
__global__ void __launch_bounds__(kThreads) cache_rows_kernel(const RowsParams p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes, kRows = kLong ? kRowsAtOnce : 1;
  constexpr int kRowBytes = CacheRow<kFmt, D>::kBytes, kSize = kF32 ? 4 : 2;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int which = blockIdx.y;
  uint32_t bh, i0;
  if constexpr (kLong) {
    bh = blockIdx.x / p.tiles;
    i0 = (blockIdx.x - bh * p.tiles) * (kGroups * kRows) + group;
  } else {
    const uint32_t r = blockIdx.x * kGroups + group;
    bh = min(r, p.rows - 1) / p.n;
    i0 = r - bh * p.n;  // p.n in a group past the last row
  }
  const uint32_t H = (uint32_t)p.c.H, b = bh / H, h = bh - b * H;
  const Strides3 xs = p.xs[which];
  uint8_t *x = p.x[which] + (b * xs.b + h * xs.h + i0 * xs.s + lane * 8) * kSize;
  const int64_t step = (int64_t)kGroups * xs.s * kSize;
  Raw<kF32> raw[kRows];
#pragma unroll
  for (int j = 0; j < kRows; ++j) raw[j] = Raw<kF32>{};
  if constexpr (kWrite && !kLong) {  // the row exists, live or not: no need to wait
    if (i0 < p.n) raw[0] = load_raw<kF32, kVec>(x);
  }
  const Span span = live_rows(p, b, i0 == 0 && lane == 0 && which == 0 && h == 0);
  const int64_t row0 = b * p.c.sb + h * p.c.sh + span.start + i0;
  uint8_t *codes = (which ? p.c.v : p.c.k) + row0 * kRowBytes + lane * (kRowBytes / kLanes);
  uint8_t *scales = (which ? p.c.v_scale : p.c.k_scale) + row0 * 4;
  bool live[kRows];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const int i = (int)i0 + j * kGroups;
    live[j] = i >= span.from && i < span.to;
    if constexpr (kWrite && kLong) {
      if (live[j]) raw[j] = load_raw<kF32, kVec>(x + j * step);
    }
  }
  if constexpr (kWrite) {
#pragma unroll
    for (int j = 0; j < kRows; ++j)
      if (__any_sync(0xffffffffu, live[j]))
        cache_store8<kFmt, kF32, kLanes>(codes + j * kGroups * kRowBytes, scales + j * kGroups * 4,
                                         lane == 0, live[j], raw[j]);
  } else {
    constexpr int kWords = kRowBytes / kLanes / 4;
    uint32_t w[kRows][kWords], scale[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const uint32_t *from = reinterpret_cast<const uint32_t *>(codes + j * kGroups * kRowBytes);
      scale[j] = 0;
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[j][k] = 0;
      if (live[j]) {
        if constexpr (kWords % 4 == 0) {
#pragma unroll
          for (int k = 0; k < kWords; k += 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(from + k);
            w[j][k] = v.x, w[j][k + 1] = v.y, w[j][k + 2] = v.z, w[j][k + 3] = v.w;
          }
        } else if constexpr (kWords == 2) {
          const uint2 v = *reinterpret_cast<const uint2 *>(from);
          w[j][0] = v.x, w[j][1] = v.y;
        } else {
          w[j][0] = *from;
        }
        if constexpr (CacheRow<kFmt, D>::kScaled)
          scale[j] = *reinterpret_cast<const uint32_t *>(scales + j * kGroups * 4);
      }
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      if (live[j] || (p.zero_rest && i0 + j * kGroups < p.n)) {
        float f[8];  // zeros where the row is not live: codes and scale are 0
        cache_values8<kFmt>(w[j], scale[j], f);
        rows_store8<kF32, kVec>(x + j * step, f);
      }
    }
  }
}

template <int kFmt, int D, bool kF32, bool kVec, bool kWrite>
cudaError_t launch_rows(RowsParams p, cudaStream_t stream) {
  constexpr uint32_t kGroups = kThreads / (D / 8), kTile = kGroups * kRowsAtOnce;
  // The long form has four rows a group in flight and its addresses and lengths
  // once a block; below half a block's rows a head it would idle.
  if (p.n >= kTile / 2) {
    p.tiles = (p.n + kTile - 1) / kTile;
    cache_rows_kernel<kFmt, D, kF32, kVec, kWrite, true>
        <<<dim3(p.rows / p.n * p.tiles, 2), kThreads, 0, stream>>>(p);
  } else {
    cache_rows_kernel<kFmt, D, kF32, kVec, kWrite, false>
        <<<dim3((p.rows + kGroups - 1) / kGroups, 2), kThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

template <int kFmt, int D, bool kWrite>
cudaError_t launch_rows_fd(const RowsParams &p, bool f32, cudaStream_t stream) {
  const int64_t m = f32 ? 4 : 8;  // elements in 16 bytes
  bool vec = true;
  for (int w = 0; w < 2; ++w)
    vec = vec && (reinterpret_cast<uintptr_t>(p.x[w]) & 15u) == 0 && p.xs[w].b % m == 0 &&
          p.xs[w].h % m == 0 && p.xs[w].s % m == 0;
  if (f32)
    return vec ? launch_rows<kFmt, D, true, true, kWrite>(p, stream)
               : launch_rows<kFmt, D, true, false, kWrite>(p, stream);
  return vec ? launch_rows<kFmt, D, false, true, kWrite>(p, stream)
             : launch_rows<kFmt, D, false, false, kWrite>(p, stream);
}

template <int kFmt, bool kWrite>
cudaError_t launch_rows_f(const RowsParams &p, bool f32, cudaStream_t stream) {
  return p.c.D == 64 ? launch_rows_fd<kFmt, 64, kWrite>(p, f32, stream)
                     : launch_rows_fd<kFmt, 128, kWrite>(p, f32, stream);
}

template <bool kWrite>
cudaError_t launch_rows_any(const CacheRowsArgs &a, const DeviceInfo &dev, cudaStream_t stream) {
  RowsParams p;
  p.c = a.c;
  p.x[0] = static_cast<uint8_t *>(a.k);
  p.x[1] = static_cast<uint8_t *>(a.v);
  p.xs[0] = a.ks;
  p.xs[1] = a.vs;
  p.n = (uint32_t)a.n;
  p.rows = (uint32_t)(a.c.B * a.c.H * a.n);  // at most 2^31 - 1
  p.tiles = 0;
  p.starts = a.starts;
  p.counts = a.counts;
  p.zero_rest = a.zero_rest;
  p.status = dev.status;
  switch (a.c.format) {
    case WFATTN_CACHE_F32: return launch_rows_f<WFATTN_CACHE_F32, kWrite>(p, a.f32, stream);
    case WFATTN_CACHE_BF16: return launch_rows_f<WFATTN_CACHE_BF16, kWrite>(p, a.f32, stream);
    case WFATTN_CACHE_E4M3: return launch_rows_f<WFATTN_CACHE_E4M3, kWrite>(p, a.f32, stream);
    default: return launch_rows_f<WFATTN_CACHE_INT4, kWrite>(p, a.f32, stream);
  }
}

// ------------------------------------------------------------------- keep

constexpr int kKeepThreads = 128;

struct KeepParams {
  CacheView c;
  const int32_t *lens, *path, *counts;
  int depth;
  int64_t path_stride;
  int32_t *new_lens;
  unsigned int *status;
};

// One block moves the K or the V rows of one head: every source row is in
// registers before the first destination is written, so the order of the path
// and rows that are both source and destination do not matter.
template <int kRowBytes>
__global__ void __launch_bounds__(kKeepThreads) cache_keep_kernel(const KeepParams p) {
  constexpr int kChunks = kRowBytes / 16;  // 16-byte pieces of a row
  constexpr int kItems = (kMaxTreeNodes * kChunks + kKeepThreads - 1) / kKeepThreads;
  __shared__ int32_t path[kMaxTreeNodes];
  const uint32_t b = blockIdx.x / (uint32_t)p.c.H, h = blockIdx.x - b * (uint32_t)p.c.H;
  const int32_t len = p.lens[b], n = p.counts ? p.counts[b] : p.depth;
  bool bad = n < 0 || n > p.depth || len < 0 || (int64_t)len + n > p.c.L;
  if (!bad && (int)threadIdx.x < n) {
    const int32_t from = p.path[b * p.path_stride + threadIdx.x];
    path[threadIdx.x] = from;
    bad = from < 0 || (int64_t)len + from >= p.c.L;
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0 && blockIdx.y == 0 && h == 0) {
    p.new_lens[b] = bad ? len : len + n;
    if (bad) atomicOr(p.status, kDevBadRowMask);
  }
  if (bad) return;
  const int64_t row0 = b * p.c.sb + h * p.c.sh + len;
  uint8_t *codes = (blockIdx.y ? p.c.v : p.c.k) + row0 * kRowBytes;
  uint32_t *scales = reinterpret_cast<uint32_t *>(blockIdx.y ? p.c.v_scale : p.c.k_scale);
  uint4 got[kItems];
  uint32_t scale = 0;
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int item = threadIdx.x + j * kKeepThreads, i = item / kChunks;
    if (i < n)
      got[j] = *reinterpret_cast<const uint4 *>(codes + (int64_t)path[i] * kRowBytes +
                                                item % kChunks * 16);
  }
  if (scales && (int)threadIdx.x < n) scale = scales[row0 + path[threadIdx.x]];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int item = threadIdx.x + j * kKeepThreads, i = item / kChunks;
    if (i < n) *reinterpret_cast<uint4 *>(codes + i * kRowBytes + item % kChunks * 16) = got[j];
  }
  if (scales && (int)threadIdx.x < n) scales[row0 + threadIdx.x] = scale;
}

}  // namespace

cudaError_t launch_cache_write(const CacheRowsArgs &a, const DeviceInfo &dev,
                               cudaStream_t stream) {
  return launch_rows_any<true>(a, dev, stream);
}

cudaError_t launch_cache_read(const CacheRowsArgs &a, const DeviceInfo &dev, cudaStream_t stream) {
  return launch_rows_any<false>(a, dev, stream);
}

cudaError_t launch_cache_keep(const CacheKeepArgs &a, const DeviceInfo &dev, cudaStream_t stream) {
  KeepParams p;
  p.c = a.c;
  p.lens = a.lens;
  p.path = a.path;
  p.counts = a.counts;
  p.depth = a.depth;
  p.path_stride = a.path_stride;
  p.new_lens = a.new_lens;
  p.status = dev.status;
  const dim3 grid((unsigned)(a.c.B * a.c.H), 2);
  switch ((a.c.format == WFATTN_CACHE_F32    ? 8
           : a.c.format == WFATTN_CACHE_BF16 ? 4
           : a.c.format == WFATTN_CACHE_E4M3 ? 2
                                             : 1) * a.c.D / 2) {
    case 32: cache_keep_kernel<32><<<grid, kKeepThreads, 0, stream>>>(p); break;
    case 64: cache_keep_kernel<64><<<grid, kKeepThreads, 0, stream>>>(p); break;
    case 128: cache_keep_kernel<128><<<grid, kKeepThreads, 0, stream>>>(p); break;
    case 256: cache_keep_kernel<256><<<grid, kKeepThreads, 0, stream>>>(p); break;
    default: cache_keep_kernel<512><<<grid, kKeepThreads, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

}  // namespace wfattn
