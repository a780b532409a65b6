// tree_decode over f32 rows with f32 queries.
#include "tree_decode_launch.cuh"

namespace wfattn {
WFATTN_TREE_DEFINE(f32_f32, WFATTN_CACHE_F32, true)
}  // namespace wfattn
