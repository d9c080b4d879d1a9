#include "linear_mma.cuh"

namespace qk {

cudaError_t launch_mma_backward_f16(int kind, const CUtensorMap &xmap, const CUtensorMap &wmap, const LinearMmaArgs &m, int grid, size_t smem, const LaunchCfg &cfg, cudaStream_t stream)
{
    return launch_mma_kind<QK_F16, true, 1>(kind, xmap, wmap, m, grid, smem, cfg, stream);
}

}  // namespace qk
