// tree_decode over bf16 rows with bf16 queries.
#include "tree_decode_launch.cuh"

namespace wfattn {
WFATTN_TREE_DEFINE(bf16_bf16, WFATTN_CACHE_BF16, false)
}  // namespace wfattn
