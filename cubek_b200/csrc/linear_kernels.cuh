// Products with quantized weights: what the kernels share.
//
//   forward    z = x W^T + b,  y = act(z) + r          x [rows, K], W [N, K], y [rows, N]
//   backward   dx = dz W,  dz = dy * act'(z),  db = sum of dz over the rows
//
// W is the tensor that dequantize returns in the type F of x (f16 or bf16): RN_F(code * RN_F(scale)).  Products are
// summed in f32 and rounded to F once, after bias, activation and residual.  With experts, W is [E, N, K] and
// the rows offsets[e] .. offsets[e + 1] of x use W[e]; rows outside every expert are neither read nor written.
#pragma once

#include "dequantize_kernels.cuh"

namespace qk {

struct LinearArgs {
    // weight: codes [E, N, K] packed along K, scales at (e / be, row / bn, col / bk) through their strides
    const uint8_t *codes;
    long long code_row, code_expert;  // bytes
    int code_align;                   // 16, 4 or 1: what base, row and expert stride are multiples of
    int n, k;
    const void *scales;
    int param;                        // QkDType of the scales
    long long scale_row, scale_col, scale_expert;  // elements
    FastDiv bn, bk;
    unsigned be;                      // experts per scale block
    int scale32;                      // 32 consecutive codes of a row (at a multiple of 32) share a scale; else 8 do
    // activations: [rows, contraction], row-major
    const void *x;
    long long x_stride;               // elements
    int rows, contraction, feats;     // forward: contraction K, features N; backward the other way round
    // output [rows, feats] and what its epilogue reads and keeps
    void *out;
    long long out_stride;
    const void *bias;
    long long bias_stride, bias_expert;
    const void *residual;
    long long residual_stride;
    void *pre;
    long long pre_stride;
    int act;                          // QkActivation
    int pairs;                        // two neighbouring features may be read and written as one 32-bit word
    // experts
    const void *offsets;              // nullptr: one expert with all rows
    int offsets64;
    int experts;
    int *error_flag;
};

// Rows of expert e.  Offsets are clamped to the tensor, so that wrong ones give wrong rows, not wrong addresses.
__device__ __forceinline__ void expert_rows(const LinearArgs &a, int e, int &lo, int &hi)
{
    if (a.offsets == nullptr) {
        lo = 0;
        hi = a.rows;
        return;
    }
    long long l, h;
    if (a.offsets64) {
        l = static_cast<const long long *>(a.offsets)[e];
        h = static_cast<const long long *>(a.offsets)[e + 1];
    } else {
        l = static_cast<const int *>(a.offsets)[e];
        h = static_cast<const int *>(a.offsets)[e + 1];
    }
    l = l < 0 ? 0 : l > a.rows ? a.rows : l;
    h = h < l ? l : h > a.rows ? a.rows : h;
    lo = (int)l;
    hi = (int)h;
}

// ---- activations, in f32 --------------------------------------------------------------------------
__device__ __forceinline__ float sigmoid_f32(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

__device__ __forceinline__ float activate(int act, float z)
{
    switch (act) {
    case QK_ACT_RELU: return z < 0.0f ? 0.0f : z;
    case QK_ACT_GELU: return 0.5f * z * erfcf(-0.70710678f * z);  // 1 + erf(t) = erfc(-t), which keeps its digits far below 0
    case QK_ACT_GELU_TANH: return z * sigmoid_f32(1.59576912f * (z + 0.044715f * z * z * z));  // (1 + tanh(t)) / 2 = sigmoid(2t)
    case QK_ACT_SILU: return z * sigmoid_f32(z);
    default: return z;
    }
}

__device__ __forceinline__ float activation_slope(int act, float z)
{
    switch (act) {
    case QK_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case QK_ACT_GELU: return 0.5f * erfcf(-0.70710678f * z) + z * 0.39894228f * __expf(-0.5f * z * z);
    case QK_ACT_GELU_TANH: {
        const float s = sigmoid_f32(1.59576912f * (z + 0.044715f * z * z * z));
        return s + z * s * (1.0f - s) * 1.59576912f * (1.0f + 0.134145f * z * z);
    }
    case QK_ACT_SILU: {
        const float s = sigmoid_f32(z);
        return s + z * s * (1.0f - s);
    }
    default: return 1.0f;
    }
}

// ---- weights ----------------------------------------------------------------------------------------
// A run of 32 consecutive codes of one weight row as it lies in memory, with its scales as stored.
template <int KIND> struct CodeRun {
    static constexpr int BITS = kind_bits(KIND);
    static constexpr int WORDS = BITS;  // 32 codes of BITS bits
    uint32_t w[WORDS];
    uint32_t s[4];  // raw scale of each 8 codes (only s[0] with scale32)
    int valid;      // codes of the run that exist (0 .. 32); the others are zero bits
};

__device__ __forceinline__ uint32_t load_scale_raw(const LinearArgs &a, long long i)
{
    return a.param == QK_F32 ? __ldg(static_cast<const uint32_t *>(a.scales) + i)
                             : (uint32_t)__ldg(static_cast<const unsigned short *>(a.scales) + i);
}
// RN_F(scale) as f32.
template <int FDT> __device__ __forceinline__ float scale_value(const LinearArgs &a, uint32_t raw)
{
    const float s = a.param == QK_F32 ? __uint_as_float(raw)
                    : a.param == QK_BF16 ? __uint_as_float(raw << 16)
                                         : __half2float(__ushort_as_half((unsigned short)raw));
    return round_to<FDT>(s);
}

// Codes row, col .. col + 31 of expert e; row and col may lie past the weight.  col is a multiple of 32.
template <int KIND> __device__ __forceinline__ void load_code_run(const LinearArgs &a, CodeRun<KIND> &r, int e, int row, int col)
{
    constexpr int BITS = CodeRun<KIND>::BITS, WORDS = CodeRun<KIND>::WORDS;
    int valid = row < a.n ? a.k - col : 0;
    valid = valid < 0 ? 0 : valid > 32 ? 32 : valid;
    r.valid = valid;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) r.w[i] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.s[i] = 0;
    if (valid == 0) return;
    const uint8_t *p = a.codes + e * a.code_expert + row * a.code_row + (long long)col * BITS / 8;
    const int bytes = (valid * BITS + 7) / 8;
    if (a.code_align == 16 && valid == 32) {
        if constexpr (WORDS == 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2 *>(p));
            r.w[0] = v.x;
            r.w[1] = v.y;
        } else {
#pragma unroll
            for (int i = 0; i < WORDS / 4; ++i) {
                const Vec16 v = ldg128_stream(p + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) r.w[4 * i + j] = v.w[j];
            }
        }
    } else if (a.code_align >= 4) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            if (4 * i + 4 <= bytes) {
                r.w[i] = __ldg(reinterpret_cast<const uint32_t *>(p) + i);
            } else {
                for (int j = 4 * i; j < bytes; ++j) r.w[i] |= (uint32_t)__ldg(p + j) << (8 * (j - 4 * i));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (4 * i + j < bytes) r.w[i] |= (uint32_t)__ldg(p + 4 * i + j) << (8 * j);
    }
    const long long s0 = (long long)(e / a.be) * a.scale_expert + (long long)fastdiv((unsigned)row, a.bn) * a.scale_row;
    if (a.scale32) {
        r.s[0] = load_scale_raw(a, s0 + (long long)fastdiv((unsigned)col, a.bk) * a.scale_col);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (8 * i < valid) r.s[i] = load_scale_raw(a, s0 + (long long)fastdiv((unsigned)(col + 8 * i), a.bk) * a.scale_col);
    }
}

// The run as 16 registers of packed F x2, in element order; what lies past the weight is +0 whatever the scale is.
template <int KIND, int FDT> __device__ __forceinline__ void decode_code_run(const LinearArgs &a, const CodeRun<KIND> &r, uint32_t *o)
{
    constexpr int WORDS = CodeRun<KIND>::WORDS, EPW = kind_elems_per_u32(KIND);
    if (a.scale32) {
        const float s = scale_value<FDT>(a, r.s[0]);
        const uint32_t s2 = h2_pack<FDT>(s, s);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) dequant_word<FDT, KIND>(r.w[i], s, s2, o + i * EPW / 2);
    } else if constexpr (EPW <= 8) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float s = scale_value<FDT>(a, r.s[g]);
            const uint32_t s2 = h2_pack<FDT>(s, s);
#pragma unroll
            for (int i = g * WORDS / 4; i < (g + 1) * WORDS / 4; ++i) dequant_word<FDT, KIND>(r.w[i], s, s2, o + i * EPW / 2);
        }
    } else {  // 16 codes a word: their blocks are multiples of 16 codes
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            const float s = scale_value<FDT>(a, r.s[2 * i]);
            dequant_word<FDT, KIND>(r.w[i], s, h2_pack<FDT>(s, s), o + i * EPW / 2);
        }
    }
    if (r.valid < 32) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (2 * i >= r.valid) o[i] = 0;
            else if (2 * i + 1 >= r.valid) o[i] &= 0xffffu;
        }
    }
}

// ---- epilogue -----------------------------------------------------------------------------------------
template <int FDT> __device__ __forceinline__ float widen_lo(uint32_t p)
{
    if constexpr (FDT == QK_BF16) return bf16_lo_to_f32(p);
    else return __low2float(*reinterpret_cast<const __half2 *>(&p));
}
template <int FDT> __device__ __forceinline__ float widen_hi(uint32_t p)
{
    if constexpr (FDT == QK_BF16) return bf16_hi_to_f32(p);
    else return __high2float(*reinterpret_cast<const __half2 *>(&p));
}

template <int FDT> __device__ __forceinline__ float load_bias(const LinearArgs &a, int e, int f)
{
    using F = typename ElemOf<FDT>::type;
    if (a.bias == nullptr || f >= a.feats) return 0.0f;
    return (float)static_cast<const F *>(a.bias)[e * a.bias_expert + f * a.bias_stride];
}

// One output element from its sum.
template <int FDT> __device__ __forceinline__ void finish_one(const LinearArgs &a, int row, int f, float sum, float bias)
{
    using F = typename ElemOf<FDT>::type;
    float z = sum + bias;
    if (a.pre) static_cast<F *>(a.pre)[row * a.pre_stride + f] = (F)z;
    z = activate(a.act, z);
    if (a.residual) z += (float)static_cast<const F *>(a.residual)[row * a.residual_stride + f];
    static_cast<F *>(a.out)[row * a.out_stride + f] = (F)z;
}

}  // namespace qk
