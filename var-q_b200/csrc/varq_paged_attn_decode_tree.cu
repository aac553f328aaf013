// The decode kernel of a paged cache for trees of drafted tokens.
#include "varq_paged_attn_decode.cuh"

namespace varq {

int paged_attn_decode_tree_run(const PagedAttnArgs& a, int rows, int splits, bool in_cluster, int tiles_per_split, float* ws_o, float* ws_ml, int* status, cudaStream_t st) {
    return launch_bits<true>(a, rows, splits, in_cluster, tiles_per_split, ws_o, ws_ml, status, st);
}

}  // namespace varq
