// Products with quantized weights for a handful of rows (single tokens, small decoding batches): bound by reading the codes.
//
// A warp multiplies 16 features with 8 or 16 rows of x over a slice of K, on mma.sync m16n8k16: the tcgen05 tiles need
// shared memory, barriers and TMEM, whose latencies a read of a few megabytes does not hide, and the work of the tensor cores
// is nothing here.  Codes go from memory to registers to the instruction: lane 4 g + t of a warp holds 32 consecutive
// codes of rows g and g + 8, and 32 consecutive elements of row g of x, at the same place t of a chunk of 128; since the
// contraction may be summed in any order, eight instructions take them four at a time from every lane as if they were in
// the instruction's order.  The warps of a CTA share K and add their sums in warp order through shared memory.
#pragma once

#include "linear_tiles.cuh"

namespace qk {

// 16 bytes (8 for 2-bit codes) times N straight to registers, or zero: no branch, so that several loads stay in flight.
template <int WORDS> __device__ __forceinline__ void load_codes_if(uint32_t *w, const uint8_t *p, uint32_t ok)
{
    if constexpr (WORDS == 2) {
        asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %3, 0;\nmov.b32 %0, 0;\nmov.b32 %1, 0;\n@p ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];\n}"
                     : "=&r"(w[0]), "=&r"(w[1])
                     : "l"(p), "r"(ok));
    } else {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4)
            asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %5, 0;\nmov.b32 %0, 0;\nmov.b32 %1, 0;\nmov.b32 %2, 0;\nmov.b32 %3, 0;\n"
                         "@p ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n}"
                         : "=&r"(w[i]), "=&r"(w[i + 1]), "=&r"(w[i + 2]), "=&r"(w[i + 3])
                         : "l"(p + 4 * i), "r"(ok));
    }
}
__device__ __forceinline__ uint32_t load_scale_if(uintptr_t at, uint32_t wide, uint32_t ok)
{
    uint32_t s;
    asm volatile("{\n.reg .pred w, h, p;\nsetp.ne.u32 p, %3, 0;\nsetp.ne.and.u32 w, %2, 0, p;\nsetp.eq.and.u32 h, %2, 0, p;\nmov.b32 %0, 0;\n"
                 "@w ld.global.nc.u32 %0, [%1];\n@h ld.global.nc.u16 %0, [%1];\n}"
                 : "=&r"(s)
                 : "l"(at), "r"(wide), "r"(ok));
    return s;
}

// A run of 32 codes of any size and alignment.
template <int KIND> __device__ __forceinline__ void fetch_run(const LinearArgs &a, CodeRun<KIND> &r, const CodeRow &row, int col)
{
    constexpr int BITS = CodeRun<KIND>::BITS, WORDS = CodeRun<KIND>::WORDS;
    const int valid = row.exists ? codes_left(a, col) : 0, bytes = (valid * BITS + 7) / 8;
    const uint8_t *p = row.codes + (long long)col * BITS / 8;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
        r.w[i] = 0;
        if (a.code_align >= 4 && 4 * i + 4 <= bytes) {
            r.w[i] = __ldg(reinterpret_cast<const uint32_t *>(p) + i);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (4 * i + j < bytes) r.w[i] |= (uint32_t)__ldg(p + 4 * i + j) << (8 * j);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r.s[i] = 0;
        if (8 * i < valid) {
            const long long at = scale_index(a, row, col + 8 * i);
            r.s[i] = a.param == QK_F32 ? __ldg(static_cast<const uint32_t *>(a.scales) + at)
                                       : (uint32_t)__ldg(static_cast<const unsigned short *>(a.scales) + at);
        }
    }
}

// 16 elements of x from `p` as packed pairs, `left` of which exist (WHOLE: all or none).
template <bool WHOLE> __device__ __forceinline__ void fetch_x(uint32_t *x, const uint16_t *p, int left)
{
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (WHOLE || left <= 8 * i || left >= 8 * i + 8) {
            const uint32_t ok = left > 8 * i;
            asm("{\n.reg .pred p;\nsetp.ne.u32 p, %5, 0;\nmov.b32 %0, 0;\nmov.b32 %1, 0;\nmov.b32 %2, 0;\nmov.b32 %3, 0;\n"
                "@p ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];\n}"
                         : "=&r"(x[4 * i]), "=&r"(x[4 * i + 1]), "=&r"(x[4 * i + 2]), "=&r"(x[4 * i + 3])
                         : "l"(p + 8 * i), "r"(ok));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = 8 * i + 2 * j;
                x[4 * i + j] = (at < left ? (uint32_t)p[at] : 0u) | (at + 1 < left ? (uint32_t)p[at + 1] << 16 : 0u);
            }
        }
    }
}

template <int FDT> __device__ __forceinline__ void mma_m16n8k16(float *d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (FDT == QK_BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int SKINNY_FEATS = 16, SKINNY_WARPS = 8;

// Whether the codes of a word are taken in the order 0, 4, 1, 5, 2, 6, 3, 7, for which x is put in the same order: fields that
// are 16 bits apart come out of a word with one shift and one logical instruction per pair.
template <int KIND, int NS> constexpr bool split_pairs = KIND == KIND_PACK4 && NS < 4;

// 16 of a run's codes (the first or the second half) as packed F x2, in element order (or the other); codes past `valid`
// are +0.  NS: scales of a run; 4: any number, and any number of codes.
template <int KIND, int FDT, int NS>
__device__ __forceinline__ void decode_half_run(const LinearArgs &a, const CodeRun<KIND> &r, int half, int valid, uint32_t *o)
{
    constexpr int WORDS = CodeRun<KIND>::WORDS / 2, EPW = kind_elems_per_u32(KIND);
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
        const uint32_t s = scale_pair<FDT>(a.param, r.s[NS == 1 ? 0 : NS == 2 ? half : 2 * half + i * EPW / 8]);
        const uint32_t w = r.w[half * WORDS + i];
        if constexpr (split_pairs<KIND, NS>) {
            constexpr uint32_t BASE = (FDT == QK_BF16) ? 0x43084308u : 0x64086408u;   // 128 or 1024, and the bias of a code
            const uint32_t bias = h2_const<FDT>(FDT == QK_BF16 ? 136.0f : 1032.0f);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[4 * i + j] = h2_mul<FDT>(h2_sub<FDT>((w >> 4 * j & 0x000F000Fu) ^ BASE, bias), s);
        } else {
            decode_word<FDT, KIND>(w, s, o + i * EPW / 2);
        }
    }
    if (NS == 4 && valid < 16 * half + 16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (16 * half + 2 * i >= valid) o[i] = 0;
            else if (16 * half + 2 * i + 1 >= valid) o[i] &= 0xffffu;
        }
    }
}

// Chunks of a warp are 8 * 128 codes apart.  Regular: aligned rows of whole runs with one or two scales, which then lie a
// constant distance apart too.
inline bool skinny_regular(const LinearArgs &a)
{
    return a.code_align == 16 && a.k % 32 == 0 && a.run_scales <= 2 && (a.scale_col == 0 || 128 * SKINNY_WARPS % a.bk.div == 0);
}

// NT: rows of x in eights.  NS: scales of a run, or 4: not regular.  A persistent CTA walks blocks of 16 features (of each
// group of rows of each expert); codes of the next ones are on their way while one is finished.
template <int KIND, int FDT, int NT, int NS>
__global__ void __launch_bounds__(32 * SKINNY_WARPS, 2) linear_skinny_kernel(const LinearMmaArgs m)
{
    constexpr int BITS = kind_bits(KIND), AHEAD = BITS == 8 ? 2 : 3, ROWS = 8 * NT;
    constexpr bool WHOLE = NS < 4;
    __shared__ float part[2][SKINNY_WARPS][ROWS][SKINNY_FEATS];
    extern __shared__ int table[];
    const LinearArgs &a = m.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
    pdl_entry();
    const MmaSchedule sched = mma_schedule(m, table, 32 * SKINNY_WARPS);
    const int first = blockIdx.x, step = gridDim.x, k = a.k, chunks = (k + 127) / 128;

    // what is fetched next.  Features past the weight read its last row; their sums are not stored.
    int ft = first, fc = warp;
    CodeRow row0 = {}, row1 = {};
    const uint8_t *p0 = nullptr, *p1 = nullptr;
    uintptr_t s0 = 0, s1 = 0;
    const uint32_t wide = a.param == QK_F32;
    const int scale_size = wide ? 4 : 2;
    const long long part_step = a.scale_col * scale_size;   // from one of a run's scales to the next
    const long long scale_step = a.scale_col ? part_step * (128 * SKINNY_WARPS / (int)a.bk.div) : 0;
    const auto enter = [&] {
        if (ft >= sched.total) return;
        const MmaTile tile = mma_tile(m, sched, ft, SKINNY_FEATS);
        row0 = code_row(a, tile.e, min(tile.f0 + g, a.n - 1));
        row1 = code_row(a, tile.e, min(tile.f0 + g + 8, a.n - 1));
        if (WHOLE) {
            const int col = fc * 128 + 32 * t4;
            p0 = row0.codes + (long long)col * BITS / 8;
            p1 = row1.codes + (long long)col * BITS / 8;
            s0 = reinterpret_cast<uintptr_t>(a.scales) + scale_index(a, row0, col) * scale_size;
            s1 = reinterpret_cast<uintptr_t>(a.scales) + scale_index(a, row1, col) * scale_size;
        }
    };
    CodeRun<KIND> q0[AHEAD], q1[AHEAD];
    const auto fetch_next = [&](int i) {
        if (ft >= sched.total || warp >= chunks) return;
        const int col = fc * 128 + 32 * t4;
        if constexpr (WHOLE) {
            const uint32_t ok = col < k;
            load_codes_if<CodeRun<KIND>::WORDS>(q0[i].w, p0, ok);
            load_codes_if<CodeRun<KIND>::WORDS>(q1[i].w, p1, ok);
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                q0[i].s[j] = load_scale_if(s0 + j * part_step, wide, ok);
                q1[i].s[j] = load_scale_if(s1 + j * part_step, wide, ok);
            }
            p0 += 16 * SKINNY_WARPS * BITS;
            p1 += 16 * SKINNY_WARPS * BITS;
            s0 += scale_step;
            s1 += scale_step;
        } else {
            fetch_run<KIND>(a, q0[i], row0, col);
            fetch_run<KIND>(a, q1[i], row1, col);
        }
        fc += SKINNY_WARPS;
        if (fc >= chunks) {
            fc = warp;
            ft += step;
            enter();
        }
    };
    enter();
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch_next(i);

    int t = first, c = warp, buf = 0;
    MmaTile tile = {};
    const uint16_t *x0[NT];
    const auto start = [&] {
        if (t >= sched.total) return;
        tile = mma_tile(m, sched, t, SKINNY_FEATS);
#pragma unroll
        for (int n = 0; n < NT; ++n) x0[n] = static_cast<const uint16_t *>(a.x) + (long long)(tile.r0 + min(8 * n + g, tile.rows - 1)) * a.x_stride + 32 * t4;
    };
    start();
    float acc[NT][4] = {};
    while (t < sched.total) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (t >= sched.total) break;
            if (c < chunks) {
                const int col = c * 128 + 32 * t4, left = WHOLE ? 32 : codes_left(a, col);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t x[NT][8], o0[8], o1[8];
#pragma unroll
                    for (int n = 0; n < NT; ++n)   // rows past the tile repeat its last one; their sums are not stored
                        fetch_x<WHOLE>(x[n], x0[n] + c * 128 + 16 * h, k - col - 16 * h);
                    if constexpr (split_pairs<KIND, NS>) {
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int j = 0; j < 8; j += 4) {
                                const uint32_t y0 = x[n][j], y1 = x[n][j + 1], y2 = x[n][j + 2], y3 = x[n][j + 3];
                                x[n][j] = __byte_perm(y0, y2, 0x5410);
                                x[n][j + 1] = __byte_perm(y0, y2, 0x7632);
                                x[n][j + 2] = __byte_perm(y1, y3, 0x5410);
                                x[n][j + 3] = __byte_perm(y1, y3, 0x7632);
                            }
                    }
                    decode_half_run<KIND, FDT, NS>(a, q0[i], h, left, o0);
                    decode_half_run<KIND, FDT, NS>(a, q1[i], h, left, o1);
                    if (h == 1) fetch_next(i);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            mma_m16n8k16<FDT>(acc[n], o0[2 * j], o1[2 * j], o0[2 * j + 1], o1[2 * j + 1], x[n][2 * j], x[n][2 * j + 1]);
                }
                c += SKINNY_WARPS;
            }
            if (c >= chunks) {
                // the warps' sums of feature g (+ 8) and rows 2 t4, 2 t4 + 1, added in warp order; the two buffers take turns, so
                // that one barrier is enough
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    part[buf][warp][8 * n + 2 * t4][g] = acc[n][0];
                    part[buf][warp][8 * n + 2 * t4 + 1][g] = acc[n][1];
                    part[buf][warp][8 * n + 2 * t4][g + 8] = acc[n][2];
                    part[buf][warp][8 * n + 2 * t4 + 1][g + 8] = acc[n][3];
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[n][j] = 0.0f;
                }
                __syncthreads();
                if ((int)threadIdx.x < ROWS * SKINNY_FEATS) {
                    const int r = threadIdx.x / SKINNY_FEATS, fi = threadIdx.x % SKINNY_FEATS, f = tile.f0 + fi;
                    if (r < tile.rows && f < a.feats) {
                        float s = part[buf][0][r][fi];
#pragma unroll
                        for (int w = 1; w < SKINNY_WARPS; ++w) s += part[buf][w][r][fi];
                        finish_one<FDT>(a, tile.r0 + r, f, s, load_bias<FDT>(a, tile.e, f));
                    }
                }
                buf ^= 1;
                t += step;
                c = warp;
                start();
            }
        }
    }
}

// ---- launch -------------------------------------------------------------------------------------------------
template <int KIND, int FDT, int NT, int NS> static cudaError_t launch_skinny_rows(const LinearArgs &a, const LaunchCfg &cfg, cudaStream_t stream)
{
    LinearMmaArgs m = {};
    m.a = a;
    m.tile_rows = 8 * NT;
    m.feat_tiles = (a.feats + SKINNY_FEATS - 1) / SKINNY_FEATS;
    m.by_feat_tiles = make_fastdiv((unsigned)m.feat_tiles);
    const bool grouped = a.offsets != nullptr;
    long long tiles = (a.rows + m.tile_rows - 1) / m.tile_rows;
    if (grouped) tiles += a.experts < a.rows ? a.experts : a.rows;   // at most
    tiles *= m.feat_tiles;
    if (tiles >= (1ll << 31)) return cudaErrorInvalidConfiguration;
    const int resident = cfg.sm_count * 2;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((unsigned)(tiles < resident ? tiles : resident));
    c.blockDim = dim3(32 * SKINNY_WARPS);
    c.dynamicSmemBytes = grouped ? (3 * a.experts + 1) * 4 : 0;
    c.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = attr;
    c.numAttrs = cfg.pdl ? 1 : 0;
    return cudaLaunchKernelEx(&c, linear_skinny_kernel<KIND, FDT, NT, NS>, m);
}

template <int KIND, int FDT> static cudaError_t launch_skinny_one(const LinearArgs &a, const LaunchCfg &cfg, cudaStream_t stream)
{
    const int scales = skinny_regular(a) ? a.run_scales : 4;
    if (a.rows <= 8 * a.experts) {
        return scales == 1 ? launch_skinny_rows<KIND, FDT, 1, 1>(a, cfg, stream) : scales == 2 ? launch_skinny_rows<KIND, FDT, 1, 2>(a, cfg, stream)
                                                                                              : launch_skinny_rows<KIND, FDT, 1, 4>(a, cfg, stream);
    }
    return scales == 1 ? launch_skinny_rows<KIND, FDT, 2, 1>(a, cfg, stream) : scales == 2 ? launch_skinny_rows<KIND, FDT, 2, 2>(a, cfg, stream)
                                                                                          : launch_skinny_rows<KIND, FDT, 2, 4>(a, cfg, stream);
}

template <int FDT> static cudaError_t launch_skinny_kind(int kind, const LinearArgs &a, const LaunchCfg &cfg, cudaStream_t stream)
{
    switch (kind) {
    case KIND_PACK8:   // bytes either way
    case KIND_I8: return launch_skinny_one<KIND_I8, FDT>(a, cfg, stream);
    case KIND_PACK4: return launch_skinny_one<KIND_PACK4, FDT>(a, cfg, stream);
    case KIND_PACK2: return launch_skinny_one<KIND_PACK2, FDT>(a, cfg, stream);
    case KIND_E2M1: return launch_skinny_one<KIND_E2M1, FDT>(a, cfg, stream);
    case KIND_E4M3: return launch_skinny_one<KIND_E4M3, FDT>(a, cfg, stream);
    case KIND_E5M2: return launch_skinny_one<KIND_E5M2, FDT>(a, cfg, stream);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace qk
