// tree_decode_sm100.cu -- attention of a tree of drafted tokens over a
// key/value cache (include/wfattn.h).
//
// One warp takes one query row (batch, head, node) and walks its keys with the
// running maximum m and sum l of an online softmax: lane i holds D/32 values of
// q and of the output, scores are shuffle sums, all in f32.
#include <math.h>

#include "cache_format.cuh"

namespace wfattn {
namespace {

constexpr int kWarps = 4;

struct TreeParams {
  CacheView c;
  int64_t rows;  // B * Hq * T
  int64_t Hq;
  int T;
  const uint8_t *q;
  uint8_t *o;
  Strides3 qs, os;
  const int32_t *lens, *counts;
  const uint64_t *tree;
  int64_t tree_stride;
  float scale_log2;
  unsigned int *status;
};

// Values d = lane*kVals .. +kVals-1 of a row.
template <int kFmt, int D>
__device__ __forceinline__ void load_vals(const uint8_t *row, const uint8_t *scale, int lane,
                                          float (&f)[D / 32]) {
  constexpr int kVals = D / 32;
  const int d0 = lane * kVals;
#pragma unroll
  for (int i = 0; i < kVals; ++i) {
    const int d = d0 + i;
    if constexpr (kFmt == WFATTN_CACHE_F32) {
      f[i] = reinterpret_cast<const float *>(row)[d];
    } else if constexpr (kFmt == WFATTN_CACHE_BF16) {
      f[i] = ptx::bf16_lo(reinterpret_cast<const uint16_t *>(row)[d]);
    } else if constexpr (kFmt == WFATTN_CACHE_E4M3) {
      f[i] = ptx::f16x2_to_f32(ptx::e4m3x2_to_f16x2(row[d])).x *
             *reinterpret_cast<const float *>(scale);
    } else {
      const uint32_t s = *reinterpret_cast<const uint32_t *>(scale);
      f[i] = fmaf(ptx::bf16_lo(s), (float)(row[d / 2] >> (4 * (d & 1)) & 15), ptx::bf16_hi(s));
    }
  }
}

template <int kFmt, int D, bool kF32>
__global__ void __launch_bounds__(32 * kWarps) tree_decode_kernel(const TreeParams p) {
  constexpr int kVals = D / 32, kRowBytes = CacheRow<kFmt, D>::kBytes;
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (r >= p.rows) return;
  const int64_t b = r / (p.Hq * p.T), hq = r / p.T % p.Hq;
  const int node = (int)(r % p.T);
  const int64_t h = hq / (p.Hq / p.c.H);
  int64_t len = p.lens[b], n = p.counts ? p.counts[b] : p.T;
  bool bad = len < 0 || n < 0 || n > p.T;
  len = len < 0 ? 0 : len;
  n = n < 0 ? 0 : n > p.T ? p.T : n;
  bad = bad || len + n > p.c.L;
  len = imin64(len, p.c.L);
  n = imin64(n, p.c.L - len);
  if (bad && lane == 0) atomicOr(p.status, kDevBadRowMask);
  const uint64_t word = p.tree ? p.tree[b * p.tree_stride + node] : (2ull << node) - 1;
  float q[kVals], acc[kVals], m = -INFINITY, l = 0.f;
  const int64_t qo = b * p.qs.b + hq * p.qs.h + node * p.qs.s + lane * kVals;
#pragma unroll
  for (int i = 0; i < kVals; ++i) {
    const float x = kF32 ? reinterpret_cast<const float *>(p.q)[qo + i]
                         : ptx::bf16_lo(reinterpret_cast<const uint16_t *>(p.q)[qo + i]);
    q[i] = x * p.scale_log2;
    acc[i] = 0.f;
  }
  const int64_t row0 = b * p.c.sb + h * p.c.sh;
  for (int64_t t = 0; node < n && t < len + n; ++t) {
    if (t >= len && !(word >> (t - len) & 1)) continue;
    float k[kVals], v[kVals];
    load_vals<kFmt, D>(p.c.k + (row0 + t) * kRowBytes, p.c.k_scale + (row0 + t) * 4, lane, k);
    load_vals<kFmt, D>(p.c.v + (row0 + t) * kRowBytes, p.c.v_scale + (row0 + t) * 4, lane, v);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kVals; ++i) s = fmaf(q[i], k[i], s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float m2 = fmaxf(m, s);
    const float f = m == -INFINITY ? 0.f : exp2f(m - m2), w = s == -INFINITY ? 0.f : exp2f(s - m2);
    l = l * f + w;
#pragma unroll
    for (int i = 0; i < kVals; ++i) acc[i] = acc[i] * f + w * v[i];
    m = m2;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t oo = b * p.os.b + hq * p.os.h + node * p.os.s + lane * kVals;
#pragma unroll
  for (int i = 0; i < kVals; ++i) {
    if constexpr (kF32)
      reinterpret_cast<float *>(p.o)[oo + i] = acc[i] * inv;
    else
      reinterpret_cast<uint16_t *>(p.o)[oo + i] =
          (uint16_t)ptx::pack_bf16x2(acc[i] * inv, 0.f);
  }
}

template <int kFmt, bool kF32>
void launch(const TreeParams &p, cudaStream_t stream) {
  const unsigned blocks = (unsigned)((p.rows + kWarps - 1) / kWarps);
  if (p.c.D == 64)
    tree_decode_kernel<kFmt, 64, kF32><<<blocks, 32 * kWarps, 0, stream>>>(p);
  else
    tree_decode_kernel<kFmt, 128, kF32><<<blocks, 32 * kWarps, 0, stream>>>(p);
}

}  // namespace

size_t tree_decode_workspace_bytes(const CacheView &, bool, int64_t, int) { return 16; }

cudaError_t launch_tree_decode(const TreeDecodeArgs &a, const DeviceInfo &dev,
                               cudaStream_t stream) {
  TreeParams p;
  p.c = a.c;
  p.rows = a.c.B * a.Hq * a.T;
  p.Hq = a.Hq;
  p.T = a.T;
  p.q = static_cast<const uint8_t *>(a.q);
  p.o = static_cast<uint8_t *>(a.o);
  p.qs = a.qs;
  p.os = a.os;
  p.lens = a.lens;
  p.counts = a.counts;
  p.tree = a.tree;
  p.tree_stride = a.tree_stride;
  p.scale_log2 = (float)((double)a.scale * 1.4426950408889634);
  p.status = dev.status;
  switch (a.c.format) {
    case WFATTN_CACHE_F32: launch<WFATTN_CACHE_F32, true>(p, stream); break;
    case WFATTN_CACHE_BF16: launch<WFATTN_CACHE_BF16, false>(p, stream); break;
    case WFATTN_CACHE_E4M3:
      a.f32 ? launch<WFATTN_CACHE_E4M3, true>(p, stream)
            : launch<WFATTN_CACHE_E4M3, false>(p, stream);
      break;
    default:
      a.f32 ? launch<WFATTN_CACHE_INT4, true>(p, stream)
            : launch<WFATTN_CACHE_INT4, false>(p, stream);
  }
  return cudaGetLastError();
}

}  // namespace wfattn
