#include "linear_wide.cuh"

namespace qk {

cudaError_t launch_wide_backward_bf16(int kind, const CUtensorMap &xmap, const CUtensorMap &wmap, const LinearMmaArgs &m, int grid, size_t smem, const LaunchCfg &cfg, cudaStream_t stream)
{
    return launch_wide_kind<QK_BF16, true>(kind, xmap, wmap, m, grid, smem, cfg, stream);
}

}  // namespace qk
