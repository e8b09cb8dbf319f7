// fast_inst_fused.cu -- instantiations of the M = 1 kernel with the fused epilogue.
#include "fast_dispatch.cuh"

namespace mcl {

mc_status_t launch_fast_fused(int wb, bool gated, const RowsArgs& a, cudaStream_t stream, bool pdl) {
    if (gated) return wb == 2 ? launch_fast_pairs<2, PRO_NONE, EPI_FUSED_GATED>(a, stream, pdl) : launch_fast_pairs<1, PRO_NONE, EPI_FUSED_GATED>(a, stream, pdl);
    return wb == 2 ? launch_fast_rows<2, PRO_NONE, EPI_FUSED>(a, stream, pdl) : launch_fast_rows<1, PRO_NONE, EPI_FUSED>(a, stream, pdl);
}

}  // namespace mcl
