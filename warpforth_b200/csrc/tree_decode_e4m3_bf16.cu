// tree_decode over e4m3 rows with bf16 queries.
#include "tree_decode_launch.cuh"

namespace wfattn {
WFATTN_TREE_DEFINE(e4m3_bf16, WFATTN_CACHE_E4M3, false)
}  // namespace wfattn
