#include "linear_skinny.cuh"

namespace qk {

cudaError_t launch_skinny_f16(int kind, const LinearArgs &a, const LaunchCfg &cfg, cudaStream_t stream) { return launch_skinny_kind<QK_F16>(kind, a, cfg, stream); }

}  // namespace qk
