// The simplest right kernel for the products with quantized weights: 64 x 64 output tiles, operands widened to f32 in
// shared memory, f32 multiply-adds.
#include "linear_kernels.cuh"

namespace qk {

template <int KIND, int FDT, bool BWD> __global__ void __launch_bounds__(256) linear_simple_kernel(const LinearArgs a)
{
    using F = typename ElemOf<FDT>::type;
    __shared__ float sw[32][65], sx[32][65];
    pdl_entry();
    const int e = blockIdx.z, f0 = blockIdx.x * 64, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    int lo, hi;
    expert_rows(a, e, lo, hi);
    for (int r0 = lo + blockIdx.y * 64; r0 < hi; r0 += gridDim.y * 64) {
        float acc[4][4] = {};
        for (int c0 = 0; c0 < a.contraction; c0 += 32) {
            const int nruns = BWD ? 64 : 64;
            if ((int)threadIdx.x < nruns) {
                CodeRun<KIND> run;
                uint32_t o[16];
                // forward: 64 weight rows of 32 columns; backward: 32 weight rows of 64 columns
                const int wr = BWD ? threadIdx.x / 2 : threadIdx.x, wc = BWD ? (threadIdx.x % 2) * 32 : 0;
                load_code_run<KIND>(a, run, e, (BWD ? c0 : f0) + wr, (BWD ? f0 : c0) + wc);
                decode_code_run<KIND, FDT>(a, run, o);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float v0 = widen_lo<FDT>(o[i]), v1 = widen_hi<FDT>(o[i]);
                    if (BWD) {
                        sw[wr][wc + 2 * i] = v0;
                        sw[wr][wc + 2 * i + 1] = v1;
                    } else {
                        sw[2 * i][wr] = v0;
                        sw[2 * i + 1][wr] = v1;
                    }
                }
            }
            for (int i = threadIdx.x; i < 64 * 32; i += 256) {
                const int r = i / 32, c = i % 32;
                sx[c][r] = (r0 + r < hi && c0 + c < a.contraction) ? (float)static_cast<const F *>(a.x)[(r0 + r) * a.x_stride + c0 + c] : 0.0f;
            }
            __syncthreads();
            const int steps = min(32, a.contraction - c0);
            for (int c = 0; c < steps; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sx[c][ty + 16 * i], sw[c][tx + 16 * j], acc[i][j]);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = r0 + ty + 16 * i, f = f0 + tx + 16 * j;
                if (r < hi && f < a.feats) finish_one<FDT>(a, r, f, acc[i][j], load_bias<FDT>(a, e, f));
            }
    }
}

template <int FDT, bool BWD> static cudaError_t launch_kind(int kind, const LinearArgs &a, const LaunchCfg &cfg, cudaStream_t stream)
{
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((unsigned)((a.feats + 63) / 64), (unsigned)min((a.rows + 63) / 64, 1024), (unsigned)a.experts);
    c.blockDim = dim3(256);
    c.stream = stream;
    switch (kind) {
    case KIND_PACK8:
    case KIND_I8: return cudaLaunchKernelEx(&c, linear_simple_kernel<KIND_I8, FDT, BWD>, a);
    case KIND_PACK4: return cudaLaunchKernelEx(&c, linear_simple_kernel<KIND_PACK4, FDT, BWD>, a);
    case KIND_PACK2: return cudaLaunchKernelEx(&c, linear_simple_kernel<KIND_PACK2, FDT, BWD>, a);
    case KIND_E2M1: return cudaLaunchKernelEx(&c, linear_simple_kernel<KIND_E2M1, FDT, BWD>, a);
    case KIND_E4M3: return cudaLaunchKernelEx(&c, linear_simple_kernel<KIND_E4M3, FDT, BWD>, a);
    case KIND_E5M2: return cudaLaunchKernelEx(&c, linear_simple_kernel<KIND_E5M2, FDT, BWD>, a);
    default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_linear_product(int fdt, int kind, bool backward, const LinearArgs &a, const LaunchCfg &cfg, cudaStream_t stream)
{
    if (fdt == QK_F16) return backward ? launch_kind<QK_F16, true>(kind, a, cfg, stream) : launch_kind<QK_F16, false>(kind, a, cfg, stream);
    return backward ? launch_kind<QK_BF16, true>(kind, a, cfg, stream) : launch_kind<QK_BF16, false>(kind, a, cfg, stream);
}

}  // namespace qk
