// Arguments that the attention kernels over a paged cache share.
#pragma once

#include "paged_common.cuh"

namespace kivi {

struct PagedAttnArgs {
    kivi_paged_layer L;
    kivi_paged_batch b;
    kivi_rows q, k, v, out;
    int q_dtype, out_dtype, n_rep, vec;
    float scale_log2;
    int pieces, chunk;           // a block's tokens are cut into pieces of `chunk` (no block has more than `pieces`)
    float *part_o, *part_ml;     // [block][KV head][piece][row]: unnormalised output, (maximum, sum)
};

#ifdef __CUDACC__
__device__ __forceinline__ void settle_args(PagedAttnArgs& a) {
    settle_paged(a.L, a.b);
    a.q.data = settled(a.q.data); a.k.data = settled(a.k.data); a.v.data = settled(a.v.data);
    a.part_o = settled(a.part_o); a.part_ml = settled(a.part_ml);
}
#endif

}  // namespace kivi
