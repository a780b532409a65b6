// tree_decode over int4 rows with bf16 queries.
#include "tree_decode_launch.cuh"

namespace wfattn {
WFATTN_TREE_DEFINE(int4_bf16, WFATTN_CACHE_INT4, false)
}  // namespace wfattn
