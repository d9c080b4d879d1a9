// dz = dy * act'(z) and the bias gradient: what the backward pass does before its product, dx = dz W.
//
// One pass over dy and z, memory bound: 2 (dy) + 2 (z) + 2 (dz) bytes per element, sums of the columns on the way.
// A CTA takes one strip of columns and one slice of an expert's rows; a column's sum is accumulated in f32 from the
// unrounded products, first per thread, then over the CTA, and where an expert has several slices their partial sums
// are added in slice order by a second small kernel: the same bits every time.
#include "linear_backward.cuh"

namespace qk {

// g *= act'(z) for N values, chosen outside the loop.  Where ReLU is flat it passes zero whatever g is: infinities and NaN of an
// overflown loss stay out.
template <int N> __device__ __forceinline__ void slope_all(int act, float *g, const float *z)
{
    if (act == QK_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = z[i] > 0.0f ? g[i] : 0.0f;
    } else if (act == QK_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] *= activation_slope(QK_ACT_SILU, z[i]);
    } else if (act == QK_ACT_GELU_TANH) {
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] *= activation_slope(QK_ACT_GELU_TANH, z[i]);
    } else if (act == QK_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] *= activation_slope(QK_ACT_GELU, z[i]);
    }
}

// VEC: elements per access.  8 row lanes of 32 threads; a strip is 32 * VEC columns.
template <int FDT, int VEC> __global__ void __launch_bounds__(256) activation_backward_kernel(const ActBackwardArgs a)
{
    using F = typename ElemOf<FDT>::type;
    __shared__ float part[8][32 * VEC];
    pdl_entry();
    const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
    const int col = (blockIdx.x * 32 + tx) * VEC, e = blockIdx.y, slice = blockIdx.z;
    LinearArgs rows = {};
    rows.offsets = a.offsets;
    rows.offsets64 = a.offsets64;
    rows.rows = a.rows;
    int lo, hi;
    expert_rows(rows, e, lo, hi);
    const int per = (hi - lo + a.slices - 1) / a.slices;
    const long long first = lo + (long long)slice * per;
    const int last = (int)min((long long)hi, first + per);
    float sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0.0f;
    constexpr int ROWS = VEC == 8 ? 4 : 2;   // rows in flight per thread
    if (col < a.n) {
        for (long long r0 = first + ty; r0 < last; r0 += 8 * ROWS) {
            float g[ROWS][VEC], z[ROWS][VEC];
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                const long long r = min(r0 + 8 * k, (long long)last - 1);
                if constexpr (VEC == 8) {
                    const Vec16 v = ldg128_stream(static_cast<const F *>(a.grad) + r * a.grad_stride + col);
                    widen16<FDT>(v, g[k]);
                    if (a.act != QK_ACT_IDENTITY) {
                        const Vec16 u = ldg128_stream(static_cast<const F *>(a.pre) + r * a.pre_stride + col);
                        widen16<FDT>(u, z[k]);
                    }
                } else {
                    g[k][0] = (float)static_cast<const F *>(a.grad)[r * a.grad_stride + col];
                    if (a.act != QK_ACT_IDENTITY) z[k][0] = (float)static_cast<const F *>(a.pre)[r * a.pre_stride + col];
                }
            }
            slope_all<ROWS * VEC>(a.act, &g[0][0], &z[0][0]);
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                const long long r = r0 + 8 * k;
                if (r >= last) break;
#pragma unroll
                for (int i = 0; i < VEC; ++i) sum[i] += g[k][i];
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    F *to = static_cast<F *>(d ? a.dz2 : a.dz);
                    if (to == nullptr) continue;
                    to += r * (d ? a.dz2_stride : a.dz_stride) + col;
                    if constexpr (VEC == 8) {
                        uint4 v;
                        v.x = h2_pack<FDT>(g[k][0], g[k][1]);
                        v.y = h2_pack<FDT>(g[k][2], g[k][3]);
                        v.z = h2_pack<FDT>(g[k][4], g[k][5]);
                        v.w = h2_pack<FDT>(g[k][6], g[k][7]);
                        *reinterpret_cast<uint4 *>(to) = v;
                    } else {
                        *to = (F)g[k][0];
                    }
                }
            }
        }
    }
    if (a.grad_bias == nullptr) return;
#pragma unroll
    for (int i = 0; i < VEC; ++i) part[ty][tx * VEC + i] = sum[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * VEC; i += 256) {
        const int c = blockIdx.x * 32 * VEC + i;
        if (c >= a.n) continue;
        float s = part[0][i];
#pragma unroll
        for (int j = 1; j < 8; ++j) s += part[j][i];
        if (a.slices > 1) a.partial[((long long)e * a.slices + slice) * a.n + c] = s;
        else static_cast<F *>(a.grad_bias)[e * a.grad_bias_expert + c * a.grad_bias_stride] = (F)s;
    }
}

template <int FDT> __global__ void __launch_bounds__(256) bias_gradient_kernel(const ActBackwardArgs a)
{
    using F = typename ElemOf<FDT>::type;
    pdl_entry();
    const int c = blockIdx.x * 256 + threadIdx.x, e = blockIdx.y;
    if (c >= a.n) return;
    float s = 0.0f;
    for (int i = 0; i < a.slices; ++i) s += a.partial[((long long)e * a.slices + i) * a.n + c];
    static_cast<F *>(a.grad_bias)[e * a.grad_bias_expert + c * a.grad_bias_stride] = (F)s;
}

// Six CTAs of strips of 256 columns for each of 148 SMs, and no slice below 32 rows of an evenly filled expert.
int bias_slices(long long rows, long long n, int experts)
{
    const long long strips = (n + 255) / 256;
    long long s = (888 + strips * experts - 1) / (strips * experts);
    const long long most = rows / (32ll * experts);
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

template <int FDT> static cudaError_t launch_dtype(const ActBackwardArgs &a, const LaunchCfg &cfg, cudaStream_t stream, int *launches)
{
    const bool vec = a.vec != 0;
    const int strip = vec ? 256 : 32;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((unsigned)((a.n + strip - 1) / strip), (unsigned)a.experts, (unsigned)a.slices);
    c.blockDim = dim3(256);
    c.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = attr;
    c.numAttrs = cfg.pdl ? 1 : 0;
    cudaError_t err = vec ? cudaLaunchKernelEx(&c, activation_backward_kernel<FDT, 8>, a) : cudaLaunchKernelEx(&c, activation_backward_kernel<FDT, 1>, a);
    *launches = 1;
    if (err != cudaSuccess || a.grad_bias == nullptr || a.slices == 1) return err;
    c.gridDim = dim3((unsigned)((a.n + 255) / 256), (unsigned)a.experts, 1);
    *launches = 2;
    return cudaLaunchKernelEx(&c, bias_gradient_kernel<FDT>, a);
}

cudaError_t launch_activation_backward(int fdt, const ActBackwardArgs &a, const LaunchCfg &cfg, cudaStream_t stream, int *launches)
{
    return fdt == QK_F16 ? launch_dtype<QK_F16>(a, cfg, stream, launches) : launch_dtype<QK_BF16>(a, cfg, stream, launches);
}

}  // namespace qk
