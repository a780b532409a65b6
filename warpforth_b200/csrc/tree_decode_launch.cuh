// tree_decode_launch.cuh -- which kernel a tree_decode call runs.
#pragma once

#include "tree_decode_wide.cuh"

namespace wfattn {
namespace tree {

// Calls f with the configuration for R query rows a cache head.  mma.sync takes
// 8 or 16 rows a warp, then pairs of warps take different rows; above 32 rows
// bf16 queries go to tcgen05, whose 128 rows cost the same however many are
// there (8 cache heads, 196122 e4m3 keys of each in two sequences, head_dim
// 128: 20 rows 119 us against 192 on tcgen05, 32 rows 123 against 192, 60 rows
// 216 against 206, 244 rows 784 against 391; 60 rows over 40134 keys of each in
// 16 sequences 70 against 83, bf16 keys 78 against 67).  f32 queries, whose products need
// more terms, stay with warps that take different rows.
template <int kFmt, bool kF32, int D, class F>
auto with_rows(int R, F f) {
  if (R <= 8) return f(Cfg<kFmt, D, kF32, 1, 1>{});
  if constexpr (kF32) {
    if (R <= 16) return f(Cfg<kFmt, D, true, 1, 2>{});
    return f(Cfg<kFmt, D, true, 1, 4>{});
  } else {
    if (R <= 16) return f(Cfg<kFmt, D, false, 2, 1>{});
    if (R <= 32) return f(Cfg<kFmt, D, false, 2, 2>{});
    return f(WideCfg<kFmt, D>{});
  }
}

template <int kFmt, bool kF32>
size_t workspace_for(int D, int R) {
  auto f = [](auto cfg) { return workspace_bytes<decltype(cfg)>(); };
  return D == 64 ? with_rows<kFmt, kF32, 64>(R, f) : with_rows<kFmt, kF32, 128>(R, f);
}

template <int kFmt, bool kF32>
cudaError_t launch_for(const Params &p, void *workspace, const DeviceInfo &dev,
                       cudaStream_t stream) {
  auto f = [&](auto cfg) {
    using C = decltype(cfg);
    if constexpr (C::kWide)
      return launch_wide<C>(p, workspace, dev, stream);
    else
      return launch<C>(p, workspace, dev, stream);
  };
  return p.c.D == 64 ? with_rows<kFmt, kF32, 64>(p.R, f) : with_rows<kFmt, kF32, 128>(p.R, f);
}

}  // namespace tree

// One translation unit a row format and query type (tree_decode_*.cu).
#define WFATTN_TREE_KINDS(X)                                                           \
  X(f32_f32, WFATTN_CACHE_F32, true) X(bf16_bf16, WFATTN_CACHE_BF16, false)            \
  X(e4m3_bf16, WFATTN_CACHE_E4M3, false) X(e4m3_f32, WFATTN_CACHE_E4M3, true)          \
  X(int4_bf16, WFATTN_CACHE_INT4, false) X(int4_f32, WFATTN_CACHE_INT4, true)
#define WFATTN_TREE_DECLARE(name, fmt, f32)                                            \
  size_t tree_workspace_##name(int D, int R);                                          \
  cudaError_t tree_launch_##name(const tree::Params &p, void *workspace,               \
                                 const DeviceInfo &dev, cudaStream_t stream);
WFATTN_TREE_KINDS(WFATTN_TREE_DECLARE)

#define WFATTN_TREE_DEFINE(name, fmt, f32)                                             \
  size_t tree_workspace_##name(int D, int R) { return tree::workspace_for<fmt, f32>(D, R); } \
  cudaError_t tree_launch_##name(const tree::Params &p, void *workspace,               \
                                 const DeviceInfo &dev, cudaStream_t stream) {         \
    return tree::launch_for<fmt, f32>(p, workspace, dev, stream);                      \
  }

}  // namespace wfattn
