#include "linear_narrow.cuh"

namespace qk {

cudaError_t launch_narrow_forward_f16(int kind, const CUtensorMap &xmap, const CUtensorMap &wmap, const LinearMmaArgs &m, int grid, size_t smem, const LaunchCfg &cfg, cudaStream_t stream)
{
    return launch_narrow_kind<QK_F16, false>(kind, xmap, wmap, m, grid, smem, cfg, stream);
}

}  // namespace qk
