// tree_decode over e4m3 rows with f32 queries.
#include "tree_decode_launch.cuh"

namespace wfattn {
WFATTN_TREE_DEFINE(e4m3_f32, WFATTN_CACHE_E4M3, true)
}  // namespace wfattn
