// cache_sm100.cu -- writing, reading and keeping rows of a key/value cache
// (formats: include/wfattn.h).
//
// All three are moves of rows: a row of D values is D/8 lanes' work, 8 values
// (16 or 32 bytes) a lane, so loads and stores are 4 to 32 bytes a lane and a
// warp touches whole 128-byte lines.  A row's maximum (e4m3) or its extremes
// (int4) are shuffles over its lanes; nothing goes through shared memory.
#include "cache_format.cuh"

namespace wfattn {
namespace {

constexpr int kThreads = 256;

struct RowsParams {
  CacheView c;
  uint8_t *x[2];          // rows of new (or read) keys, values
  Strides3 xs[2];         // element strides
  uint32_t n, rows;       // rows a head, rows in all
  const int32_t *starts, *counts;
  bool zero_rest;
  unsigned int *status;
};

// The 8 values x[0..7] of the caller's rows as f32.  kVec: 16-byte aligned.
template <bool kF32, bool kVec>
__device__ __forceinline__ void rows_load8(const uint8_t *x, float (&f)[8]) {
  if constexpr (kF32 && kVec) {
    cache_load8<WFATTN_CACHE_F32>(x, 0, f);
  } else if constexpr (kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = reinterpret_cast<const float *>(x)[i];
  } else if constexpr (kVec) {
    cache_load8<WFATTN_CACHE_BF16>(x, 0, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(x)[i] << 16);
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
template <int kFmt, int kLanes>
__device__ __forceinline__ void cache_store8(uint8_t *codes, uint8_t *scale, bool first, bool live,
                                             const float (&f)[8]) {
  if constexpr (kFmt == WFATTN_CACHE_F32) {
    if (live) rows_store8<true, true>(codes, f);
  } else if constexpr (kFmt == WFATTN_CACHE_BF16) {
    if (live) rows_store8<false, true>(codes, f);
  } else {
    // |x| as an integer orders like |x|; infinities and NaN are the largest
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
#pragma unroll
    for (int m = 1; m < kLanes; m <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
    bool bad = top >= 0x7f800000u;
    if constexpr (kFmt == WFATTN_CACHE_E4M3) {
      // 448 = 1.75 * 2^8: the exponent of the smallest 2^e with |x| <= 448 2^e
      const int e = max((int)(top >> 23) - 135 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
      const float inv = bad ? 0.f : __uint_as_float((uint32_t)(127 - e) << 23);
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
      float lo = f[0], hi = f[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) lo = fminf(lo, f[i]), hi = fmaxf(hi, f[i]);
#pragma unroll
      for (int m = 1; m < kLanes; m <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
      }
      const float m = to_bf16_directed<true>(lo);
      const float s = to_bf16_directed<false>(__fdiv_rn(__fsub_rn(hi, m), 15.f));
      bad = bad || !(s <= 3.38953139e38f);  // the largest bf16
      uint32_t w = 0;
      if (!bad && s > 0.f) {
        // rint(fl(a / s)): a * (1 / s) is within 4 ulp of it, so only values
        // next to a half need the division itself
        const float inv = __frcp_rn(s);
        float r[8];
        bool near_half = inv > 1e38f;  // 1 / s overflows
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a = __fsub_rn(f[i], m), y = a * inv;
          r[i] = rintf(y);
          near_half = near_half || fabsf(fabsf(y - r[i]) - 0.5f) < 1e-5f;
        }
        if (near_half) {
#pragma unroll
          for (int i = 0; i < 8; ++i) r[i] = rintf(__fdiv_rn(__fsub_rn(f[i], m), s));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) w |= (uint32_t)fminf(fmaxf(r[i], 0.f), 15.f) << (4 * i);
      }
      if (!live) return;
      *reinterpret_cast<uint32_t *>(codes) = w;
      if (first)
        *reinterpret_cast<uint32_t *>(scale) =
            bad ? 0x7fc07fc0u : (__float_as_uint(s) >> 16) | (__float_as_uint(m) & 0xffff0000u);
    }
  }
}

// Where the caller's row r of one head lies in the cache (-1: not live).
__device__ __forceinline__ int64_t cache_row(const RowsParams &p, uint32_t bh, uint32_t i,
                                             int64_t b, bool report) {
  int32_t n = p.counts ? p.counts[b] : (int32_t)p.n;
  const int64_t at = (int64_t)p.starts[b] + i;
  bool bad = n < 0 || n > (int32_t)p.n;
  n = n > (int32_t)p.n ? (int32_t)p.n : n;
  const bool live = (int32_t)i < n;
  const bool inside = at >= 0 && at < p.c.L;
  if (report && (bad || (live && !inside))) atomicOr(p.status, kDevBadRowMask);
  const int64_t h = bh - b * p.c.H;
  return live && inside ? b * p.c.sb + h * p.c.sh + at : -1;
}

// One row (of K or of V) a lane group, kRows of them one after the other.
template <int kFmt, int D, bool kF32, bool kVec, bool kWrite, int kRows>
__global__ void __launch_bounds__(kThreads) cache_rows_kernel(const RowsParams p) {
  constexpr int kLanes = D / 8, kGroups = kThreads / kLanes;
  constexpr int kRowBytes = CacheRow<kFmt, D>::kBytes;
  const int which = blockIdx.y, lane = threadIdx.x % kLanes;
  uint8_t *codes = which ? p.c.v : p.c.k;
  uint8_t *scales = which ? p.c.v_scale : p.c.k_scale;
  const Strides3 xs = p.xs[which];
  int64_t row[kRows];
  uint8_t *x[kRows];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    const uint32_t r = (blockIdx.x * kRows + j) * kGroups + threadIdx.x / kLanes;
    row[j] = -1;
    x[j] = nullptr;
    if (r < p.rows) {
      const uint32_t bh = r / p.n, i = r - bh * p.n;
      const uint32_t b = bh / (uint32_t)p.c.H;
      row[j] = cache_row(p, bh, i, b, lane == 0 && which == 0);
      x[j] = p.x[which] + (b * xs.b + (int64_t)(bh - b * (uint32_t)p.c.H) * xs.h + i * xs.s +
                           lane * 8) * (kF32 ? 4 : 2);
    }
  }
  float f[kRows][8];
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[j][e] = 0.f;
    if (row[j] >= 0) {
      if constexpr (kWrite) {
        rows_load8<kF32, kVec>(x[j], f[j]);
      } else {
        const uint32_t s = CacheRow<kFmt, D>::kScaled
                               ? *reinterpret_cast<const uint32_t *>(scales + row[j] * 4)
                               : 0u;
        cache_load8<kFmt>(codes + row[j] * kRowBytes + lane * (kRowBytes / kLanes), s, f[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kRows; ++j) {
    if constexpr (kWrite)
      cache_store8<kFmt, kLanes>(codes + row[j] * kRowBytes + lane * (kRowBytes / kLanes),
                                 scales + row[j] * 4, lane == 0, row[j] >= 0, f[j]);
    else if (row[j] >= 0 || (p.zero_rest && x[j]))
      rows_store8<kF32, kVec>(x[j], f[j]);
  }
}

template <int kFmt, int D, bool kF32, bool kVec, bool kWrite>
cudaError_t launch_rows(const RowsParams &p, const DeviceInfo &dev, cudaStream_t stream) {
  constexpr uint32_t kGroups = kThreads / (D / 8);
  // One row a group keeps every SM busy on few rows; with rows for four full
  // waves, four a group keep four times the bytes in flight.
  const uint32_t blocks = (p.rows + kGroups - 1) / kGroups;
  if (blocks < 32u * (uint32_t)dev.sm_count)
    cache_rows_kernel<kFmt, D, kF32, kVec, kWrite, 1><<<dim3(blocks, 2), kThreads, 0, stream>>>(p);
  else
    cache_rows_kernel<kFmt, D, kF32, kVec, kWrite, 4>
        <<<dim3((blocks + 3) / 4, 2), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <int kFmt, int D, bool kWrite>
cudaError_t launch_rows_fd(const RowsParams &p, bool f32, const DeviceInfo &dev,
                           cudaStream_t stream) {
  const int64_t m = f32 ? 4 : 8;  // elements in 16 bytes
  bool vec = true;
  for (int w = 0; w < 2; ++w)
    vec = vec && (reinterpret_cast<uintptr_t>(p.x[w]) & 15u) == 0 && p.xs[w].b % m == 0 &&
          p.xs[w].h % m == 0 && p.xs[w].s % m == 0;
  if (f32)
    return vec ? launch_rows<kFmt, D, true, true, kWrite>(p, dev, stream)
               : launch_rows<kFmt, D, true, false, kWrite>(p, dev, stream);
  return vec ? launch_rows<kFmt, D, false, true, kWrite>(p, dev, stream)
             : launch_rows<kFmt, D, false, false, kWrite>(p, dev, stream);
}

template <int kFmt, bool kWrite>
cudaError_t launch_rows_f(const RowsParams &p, bool f32, const DeviceInfo &dev,
                          cudaStream_t stream) {
  return p.c.D == 64 ? launch_rows_fd<kFmt, 64, kWrite>(p, f32, dev, stream)
                     : launch_rows_fd<kFmt, 128, kWrite>(p, f32, dev, stream);
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
  p.starts = a.starts;
  p.counts = a.counts;
  p.zero_rest = a.zero_rest;
  p.status = dev.status;
  switch (a.c.format) {
    case WFATTN_CACHE_F32: return launch_rows_f<WFATTN_CACHE_F32, kWrite>(p, a.f32, dev, stream);
    case WFATTN_CACHE_BF16: return launch_rows_f<WFATTN_CACHE_BF16, kWrite>(p, a.f32, dev, stream);
    case WFATTN_CACHE_E4M3: return launch_rows_f<WFATTN_CACHE_E4M3, kWrite>(p, a.f32, dev, stream);
    default: return launch_rows_f<WFATTN_CACHE_INT4, kWrite>(p, a.f32, dev, stream);
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
