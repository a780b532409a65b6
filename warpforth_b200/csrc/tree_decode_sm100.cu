// tree_decode_sm100.cu -- attention of a tree of drafted tokens over a
// key/value cache: choice of the kernel (tree_decode_launch.cuh) by row format and
// query type.
#include "tree_decode_launch.cuh"

namespace wfattn {

size_t tree_decode_workspace_bytes(const CacheView &c, bool f32, int64_t Hq, int T) {
  const int R = (int)(Hq / c.H * T);  // at most kMaxTreeRows
#define WFATTN_TREE_CASE(name, fmt, is_f32) \
  if (c.format == fmt && f32 == is_f32) return tree_workspace_##name(c.D, R);
  WFATTN_TREE_KINDS(WFATTN_TREE_CASE)
#undef WFATTN_TREE_CASE
  return 0;
}

cudaError_t launch_tree_decode(const TreeDecodeArgs &a, const DeviceInfo &dev,
                               cudaStream_t stream) {
  tree::Params p;
  p.c = a.c;
  p.G = (int)(a.Hq / a.c.H);
  p.T = a.T;
  p.R = p.G * p.T;  // at most kMaxTreeRows
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
#define WFATTN_TREE_CASE(name, fmt, is_f32) \
  if (a.c.format == fmt && a.f32 == is_f32) return tree_launch_##name(p, a.workspace, dev, stream);
  WFATTN_TREE_KINDS(WFATTN_TREE_CASE)
#undef WFATTN_TREE_CASE
  return cudaErrorInvalidValue;
}

}  // namespace wfattn
