// tree_decode over int4 rows with f32 queries.
#include "tree_decode_launch.cuh"

namespace wfattn {
WFATTN_TREE_DEFINE(int4_f32, WFATTN_CACHE_INT4, true)
}  // namespace wfattn
