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
    int run_scales;                   // scales of 32 consecutive codes of a row (at a multiple of 32): 1, 2 or 4
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
    int pairs;                        // two neighbouring features may be read and written as one 32-bit word,
    int wide;                         // 16 of them as 32 bytes (32) or twice 16 (16); 0: neither
    // experts
    const void *offsets;              // nullptr: one expert with all rows
    int offsets64;
    int experts;
    int *error_flag;
};

// Rows of expert e; returns whether its offsets descend.  They are clamped to the tensor, so that wrong ones give wrong rows,
// not wrong addresses.
__device__ __forceinline__ bool expert_rows(const LinearArgs &a, int e, int &lo, int &hi)
{
    if (a.offsets == nullptr) {
        lo = 0;
        hi = a.rows;
        return false;
    }
    long long l, h;
    if (a.offsets64) {
        l = static_cast<const long long *>(a.offsets)[e];
        h = static_cast<const long long *>(a.offsets)[e + 1];
    } else {
        l = static_cast<const int *>(a.offsets)[e];
        h = static_cast<const int *>(a.offsets)[e + 1];
    }
    const bool descend = h < l;
    l = l < 0 ? 0 : l > a.rows ? a.rows : l;
    h = h < l ? l : h > a.rows ? a.rows : h;
    lo = (int)l;
    hi = (int)h;
    return descend;
}

// ---- activations, in f32 --------------------------------------------------------------------------
__device__ __forceinline__ float sigmoid_f32(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// The normal distribution Phi(z), and exp(-z^2 / 2) on the way.  With x = |z| / sqrt(2) and t = 1 / (1 + 0.3275911 x), the form
// of Abramowitz and Stegun 7.1.26, erfc(x) = exp(-x^2) t P(t); P of degree 7 was fitted here to the smallest relative error
// over x in [0, 9.5]: 1.1e-7, 5e-7 with the f32 roundings of t and P.  A third of the instructions of erfcf.
__device__ __forceinline__ float normal_cdf(float z, float &bell)
{
    const float t = __fdividef(1.0f, fmaf(0.3275911f * 0.70710678f, fabsf(z), 1.0f));
    bell = __expf(-0.5f * z * z);
    float p = -0.141663104f;
    p = fmaf(p, t, 0.498880595f);
    p = fmaf(p, t, -0.409603357f);
    p = fmaf(p, t, 0.456564605f);
    p = fmaf(p, t, 0.023715185f);
    p = fmaf(p, t, 0.206398115f);
    p = fmaf(p, t, 0.180649981f);
    p = fmaf(p, t, 0.185058087f);
    const float tail = 0.5f * bell * t * p;
    return z < 0.0f ? tail : 1.0f - tail;
}

__device__ __forceinline__ float activate(int act, float z)
{
    switch (act) {
    case QK_ACT_RELU: return z < 0.0f ? 0.0f : z;
    case QK_ACT_GELU: {
        float bell;
        return z * normal_cdf(z, bell);
    }
    case QK_ACT_GELU_TANH: return z * sigmoid_f32(1.59576912f * (z + 0.044715f * z * z * z));  // (1 + tanh(t)) / 2 = sigmoid(2t)
    case QK_ACT_SILU: return z * sigmoid_f32(z);
    default: return z;
    }
}

__device__ __forceinline__ float activation_slope(int act, float z)
{
    switch (act) {
    case QK_ACT_GELU: {
        float bell;
        const float cdf = normal_cdf(z, bell);
        return cdf + z * 0.39894228f * bell;
    }
    case QK_ACT_GELU_TANH: {
        const float s = sigmoid_f32(1.59576912f * (z + 0.044715f * z * z * z));
        return s + z * s * (1.0f - s) * 1.59576912f * (1.0f + 0.134145f * fminf(z * z, 1e30f));   // s (1 - s) is zero long before: no 0 inf
    }
    case QK_ACT_SILU: {
        const float s = sigmoid_f32(z);
        return s + z * s * (1.0f - s);
    }
    default: return 1.0f;
    }
}

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

// ---- weights ----------------------------------------------------------------------------------------
// A run of 32 consecutive codes of one weight row, at a column that is a multiple of 32, with its scales as stored.
template <int KIND> struct CodeRun {
    static constexpr int BITS = kind_bits(KIND);
    static constexpr int WORDS = BITS;  // 32 codes of BITS bits
    uint32_t w[WORDS];
    uint32_t s[4];  // raw scales of equal parts
};

// A weight row: its codes and its scales.
struct CodeRow {
    const uint8_t *codes;
    long long scale;  // index of its first scale
    int exists;
};

__device__ __forceinline__ CodeRow code_row(const LinearArgs &a, int e, int row)
{
    CodeRow c;
    c.codes = a.codes + e * a.code_expert + row * a.code_row;
    c.scale = (long long)fastdiv((unsigned)row, a.bn) * a.scale_row;
    if (e > 0) c.scale += (long long)(a.be == 1 ? e : e / (int)a.be) * a.scale_expert;
    c.exists = row < a.n;
    return c;
}

__device__ __forceinline__ int codes_left(const LinearArgs &a, int col)
{
    const int left = a.k - col;
    return left < 0 ? 0 : left > 32 ? 32 : left;
}

__device__ __forceinline__ long long scale_index(const LinearArgs &a, const CodeRow &row, int col)
{
    return row.scale + (long long)fastdiv((unsigned)col, a.bk) * a.scale_col;
}

// RN_F(scale) as packed F x2, both halves.
template <int FDT> __device__ __forceinline__ uint32_t scale_pair(int param, uint32_t raw)
{
    if (param == FDT) return raw * 0x10001u;
    if (param == QK_F32) return h2_pack<FDT>(__uint_as_float(raw), __uint_as_float(raw));
    const float s = param == QK_BF16 ? __uint_as_float(raw << 16) : __half2float(__ushort_as_half((unsigned short)raw));
    return h2_pack<FDT>(s, s);
}

// One stored word times its scale, as packed F x2 in element order: dequant_word itself, so that the weight is dequantize's to
// the bit for every scale.  (8-bit codes in bf16 from one multiply-add, (32768 + b) s - 32896 s, is 0.5 to 2 % faster, 6 % where
// pairs of CTAs wait for the weight - 16 rows of 14336 x 4096 33.5 us, here 34.0; 4096 rows 428 and 429; 8 experts of 160 rows
// 309 and 328 - but 32896 s is no finite f32 from |s| = 2^113 on.  One step or two, by each run's scales: 34.7 and 319.)
template <int FDT, int KIND> __device__ __forceinline__ void decode_word(uint32_t w, uint32_t s2, uint32_t *o)
{
    dequant_word<FDT, KIND>(w, widen_lo<FDT>(s2), s2, o);
}

// The run as 16 registers of packed F x2, in element order; codes past `valid` are +0 whatever the scale is.
// NS: scales of a run (1, 2 or 4).  WHOLE: all 32 codes exist.
template <int KIND, int FDT, int NS, bool WHOLE>
__device__ __forceinline__ void decode_code_run(const LinearArgs &a, const CodeRun<KIND> &r, int valid, uint32_t *o)
{
    constexpr int WORDS = CodeRun<KIND>::WORDS, EPW = kind_elems_per_u32(KIND);
    uint32_t s[NS];
#pragma unroll
    for (int g = 0; g < NS; ++g) s[g] = scale_pair<FDT>(a.param, r.s[g]);
#pragma unroll
    for (int i = 0; i < WORDS; ++i) decode_word<FDT, KIND>(r.w[i], s[i * EPW * NS / 32], o + i * EPW / 2);
    if (!WHOLE && valid < 32) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (2 * i >= valid) o[i] = 0;
            else if (2 * i + 1 >= valid) o[i] &= 0xffffu;
        }
    }
}

// Runs on their way from memory where they cannot be fetched as tiles: a thread copies its own ones to its own places in
// shared memory by asynchronous copies of 16, 8 or 4 bytes, several steps ahead, and nothing but the thread itself waits for
// them.  Rows that start on no word are copied with the words that hold them, one more than a run has.
template <int KIND> struct StagedRuns {
    static constexpr int WORDS = CodeRun<KIND>::WORDS;
    static constexpr int AHEAD = WORDS >= 4 ? 2 : 3;
    __host__ __device__ static constexpr int slot_bytes(int threads) { return threads * (WORDS * 4 + 20); }
};

__device__ __forceinline__ void copy_async16(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async8(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Starts the copy of codes col .. col + 31 into the slot at shared address `slot` (thread `id` of `threads`); what lies past
// the weight becomes zero bits.  Scales of 16 bits are copied with the aligned word that holds them.
template <int KIND>
__device__ __forceinline__ void stage_code_run(const LinearArgs &a, uint32_t slot, int id, int threads, const CodeRow &row, int col)
{
    constexpr int BITS = CodeRun<KIND>::BITS, WORDS = CodeRun<KIND>::WORDS;
    const int valid = row.exists ? codes_left(a, col) : 0;
    const int bytes = (valid * BITS + 7) / 8;
    const uint8_t *p = valid ? row.codes + (long long)col * BITS / 8 : a.codes;
    if (a.code_align == 16) {
        if constexpr (WORDS == 2) {
            copy_async8(slot + id * 8, p, bytes);
        } else {
#pragma unroll
            for (int i = 0; i < WORDS / 4; ++i) {
                const int left = bytes - 16 * i;
                copy_async16(slot + (i * threads + id) * 16, left > 0 ? p + 16 * i : a.codes, left < 0 ? 0 : left > 16 ? 16 : left);
            }
        }
    } else {
        const uintptr_t word = reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3, none = reinterpret_cast<uintptr_t>(a.codes) & ~(uintptr_t)3;
        const int span = valid ? (int)(reinterpret_cast<uintptr_t>(p) - word) + bytes : 0;   // bytes from the first word to the run's end
#pragma unroll
        for (int i = 0; i <= WORDS; ++i) {
            const uint32_t dst = i == WORDS ? slot + threads * (WORDS * 4 + 16) + id * 4
                                            : WORDS == 2 ? slot + id * 8 + i * 4 : slot + ((i / 4) * threads + id) * 16 + (i % 4) * 4;
            if (i < WORDS || a.code_align < 4) copy_async4(dst, reinterpret_cast<const void *>(span > 4 * i ? word + 4 * i : none), span > 4 * i ? 4 : 0);
        }
    }
    const uint32_t scales = slot + threads * WORDS * 4 + id * 4;
    const int part = 32 / a.run_scales;   // codes of a scale
#pragma unroll 1
    for (int i = 0; i < a.run_scales; ++i) {
        const bool take = part * i < valid;
        const long long at = take ? scale_index(a, row, col + part * i) : 0;
        const uintptr_t q = reinterpret_cast<uintptr_t>(a.scales) + (a.param == QK_F32 ? at * 4 : at * 2);
        copy_async4(scales + i * threads * 4, reinterpret_cast<const void *>(q & ~(uintptr_t)3), take ? 4 : 0);
    }
}

// The codes of a staged run, once its copies have arrived; it starts `skip` bytes into its first word.
template <int KIND> __device__ __forceinline__ void take_codes(CodeRun<KIND> &r, uint32_t slot, int id, int threads, unsigned skip)
{
    constexpr int WORDS = CodeRun<KIND>::WORDS;
    if constexpr (WORDS == 2) {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "r"(slot + id * 8) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(r.w[i]), "=r"(r.w[i + 1]), "=r"(r.w[i + 2]), "=r"(r.w[i + 3])
                         : "r"(slot + (i / 4 * threads + id) * 16)
                         : "memory");
    }
    if (skip != 0) {
        uint32_t last;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(last) : "r"(slot + threads * (WORDS * 4 + 16) + id * 4) : "memory");
#pragma unroll
        for (int i = 0; i < WORDS; ++i) r.w[i] = __funnelshift_r(r.w[i], i + 1 < WORDS ? r.w[i + 1] : last, 8 * skip);
    }
}
// A scale staged at shared address `from`; `at`: its address in memory (of which the last bits say where in the word it is).
__device__ __forceinline__ uint32_t take_scale(const LinearArgs &a, uint32_t from, unsigned at)
{
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
    return a.param == QK_F32 ? v : at & 2 ? v >> 16 : v & 0xffffu;
}

// ---- epilogue -----------------------------------------------------------------------------------------
template <int FDT> __device__ __forceinline__ float load_bias(const LinearArgs &a, int e, int f)
{
    using F = typename ElemOf<FDT>::type;
    if (a.bias == nullptr || f >= a.feats) return 0.0f;
    return (float)static_cast<const F *>(a.bias)[e * a.bias_expert + f * a.bias_stride];
}

// The activation of N values, chosen outside the loop: one activation's code is fetched, not all of them N times.
template <int N> __device__ __forceinline__ void activate_all(int act, float *z)
{
    if (act == QK_ACT_IDENTITY) return;
    if (act == QK_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = activate(QK_ACT_RELU, z[i]);
    } else if (act == QK_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = activate(QK_ACT_SILU, z[i]);
    } else if (act == QK_ACT_GELU_TANH) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = activate(QK_ACT_GELU_TANH, z[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = activate(QK_ACT_GELU, z[i]);
    }
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
