// Products with quantized weights for a handful of rows (single tokens, small decoding batches): bound by reading the codes.
//
// A warp multiplies 16 or 32 features with 8 rows of x over a slice of K, on mma.sync m16n8k16: the tcgen05 tiles need
// shared memory, barriers and TMEM, whose latencies a read of a few megabytes does not hide, and the work of the tensor cores
// is nothing here.  Lane 4 g + t of a warp takes 32 consecutive codes of rows g and g + 8, and 32 consecutive elements of row g
// of x, at the same place t of a chunk of 128; since the contraction may be summed in any order, eight instructions take
// them four at a time from every lane as if they were in the instruction's order.  Groups of 2, 4 or 8 warps share K and
// add their sums in warp order through shared memory.
// Codes are on their way two chunks ahead, by asynchronous copies into the warp's own ring in shared memory: whole rows of a
// chunk at a time, and no registers, so that 24 warps fit an SM (with a ring in registers 16 did: 127 us for 206 MB of
// 4-bit codes of 7 experts, 85 now).
#pragma once

#include "linear_tiles.cuh"

namespace qk {

// A run of 32 codes of any size and alignment, straight to registers.
template <int KIND> __device__ __forceinline__ void fetch_run(const LinearArgs &a, CodeRun<KIND> &r, const CodeRow &row, int col)
{
    constexpr int BITS = CodeRun<KIND>::BITS, WORDS = CodeRun<KIND>::WORDS;
    // the words that hold the run, and what lies in them before it shifted out
    const int valid = row.exists ? codes_left(a, col) : 0, bytes = (valid * BITS + 7) / 8;
    const uintptr_t p = reinterpret_cast<uintptr_t>(row.codes) + (long long)col * BITS / 8, word = p & ~(uintptr_t)3;
    const unsigned skip = (unsigned)(p - word);
    uint32_t raw[WORDS + 1];
#pragma unroll
    for (int i = 0; i <= WORDS; ++i)
        raw[i] = valid && (int)skip + bytes > 4 * i ? __ldg(reinterpret_cast<const uint32_t *>(word) + i) : 0u;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) r.w[i] = __funnelshift_r(raw[i], raw[i + 1], 8 * skip);
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
            asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %5, 0;\nmov.b32 %0, 0;\nmov.b32 %1, 0;\nmov.b32 %2, 0;\nmov.b32 %3, 0;\n"
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

constexpr int SKINNY_FEATS = 16, SKINNY_ROWS = 8, SKINNY_WARPS = 8;

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

// Regular: aligned rows of whole runs with one or two scales, which then lie a constant distance, whole words, apart from one
// of a warp's chunks (at least 2 * 128 codes apart) to the next, an expert's within 2 GiB.
inline bool skinny_regular(const LinearArgs &a)
{
    const double extent = ((a.n - 1) / (double)a.bn.div * a.scale_row + (a.k - 1) / (double)a.bk.div * a.scale_col + 1) * 4;
    return a.code_align == 16 && a.k % 32 == 0 && a.run_scales <= 2 && (a.scale_col == 0 || 128 % a.bk.div == 0) && extent < 2e9;
}

constexpr int SKINNY_SLOTS = 3;
// Shared memory: a ring per warp, and the warps' sums.
__host__ __device__ constexpr int skinny_ring_bytes(int bits, int r, int ns) { return SKINNY_SLOTS * r * (256 * bits + 256 * ns); }
__host__ __device__ constexpr int skinny_bytes(int bits, int r, int ns)
{
    return SKINNY_WARPS * ((ns < 4 ? skinny_ring_bytes(bits, r, ns) : 0) + SKINNY_ROWS * SKINNY_FEATS * r * 4);
}

// R: features of a block in sixteens.  NS: scales of a run, or 4: not regular.  A persistent CTA walks
// blocks of features (of each group of rows of each expert); codes of the next ones are on their way while one is finished.
// `split`: warps that share a block's K.
template <int KIND, int FDT, int R, int NS>
__global__ void __launch_bounds__(32 * SKINNY_WARPS, NS < 4 ? 3 : 2) linear_skinny_kernel(const LinearMmaArgs m)
{
    constexpr int BITS = kind_bits(KIND), ROWS = SKINNY_ROWS, FEATS = SKINNY_FEATS * R, AHEAD = SKINNY_SLOTS - 1;
    constexpr bool WHOLE = NS < 4;
    constexpr uint32_t CODES = R * 256 * BITS, SLOT = CODES + R * 256 * NS;   // 16 R rows of 128 codes, and their scales
    extern __shared__ __align__(128) uint8_t dyn[];
    const LinearArgs &a = m.a;
    const int lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
    const int share = m.split, group = threadIdx.x / 32 / share, warp = threadIdx.x / 32 % share;   // warp of the group
    float *part = reinterpret_cast<float *>(dyn + (WHOLE ? SKINNY_WARPS * skinny_ring_bytes(BITS, R, NS) : 0)) +
                  group * share * ROWS * FEATS;   // [warp][row][feature]
    const auto meet = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * share) : "memory"); };
    pdl_entry();
    const MmaSchedule sched = mma_schedule(m, reinterpret_cast<int *>(dyn + skinny_bytes(BITS, R, NS)), 32 * SKINNY_WARPS);
    const int groups = SKINNY_WARPS / share, first = blockIdx.x * groups + group, step = gridDim.x * groups, k = a.k, chunks = (k + 127) / 128;
    const uint32_t wide = a.param == QK_F32;
    const int scale_size = wide ? 4 : 2;
    const int part_step = (int)a.scale_col * scale_size;   // bytes from one of a run's scales to the next
    const int scale_step = a.scale_col ? part_step * (128 * share / (int)a.bk.div) : 0;
    const auto expert_scales = [&](int e) {
        return reinterpret_cast<uintptr_t>(a.scales) + (long long)(a.be == 1 ? e : e / (int)a.be) * a.scale_expert * scale_size;
    };
    const auto scale_offset = [&](int f) {   // from there, of chunk `warp`
        return (int)(fastdiv((unsigned)min(f, a.n - 1), a.bn) * a.scale_row + fastdiv((unsigned)(warp * 128 + 32 * t4), a.bk) * a.scale_col) * scale_size;
    };

    // What is copied next.  A lane copies one piece of 16 bytes of every ROWS_AT_ONCE-th row, so that neighbouring lanes copy
    // neighbouring pieces.
    constexpr int PIECES = BITS, ROWS_AT_ONCE = 32 / PIECES, COPIES = 16 * R / ROWS_AT_ONCE;   // 128 codes are BITS pieces
    const int piece = lane % PIECES, copy_row = lane / PIECES;
    const uint32_t ring = smem_u32(dyn) + threadIdx.x / 32 * skinny_ring_bytes(BITS, R, NS), ring_end = ring + SKINNY_SLOTS * SLOT;
    uint32_t in = ring, out = ring;
    int ft = first, fc = warp;
    const uint8_t *from = nullptr;
    const long long row_step = ROWS_AT_ONCE * a.code_row;
    uintptr_t scales = 0;
    int scale_from[WHOLE ? 2 * R : 1], rows_left = 0;
    const auto enter = [&] {
        if (ft >= sched.total) return;
        const MmaTile tile = mma_tile(m, sched, ft, FEATS);
        from = a.codes + tile.e * a.code_expert + (tile.f0 + copy_row) * a.code_row + warp * 16 * BITS + piece * 16;
        rows_left = a.n - tile.f0 - copy_row;
        scales = expert_scales(tile.e);
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) scale_from[i] = scale_offset(tile.f0 + 8 * i + g);
    };
    const auto copy_next = [&] {
        if (ft < sched.total && warp < chunks) {
            const bool exists = fc * 128 + piece * (128 / PIECES) < k;   // runs of 32 codes exist wholly or not
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
                const int row = copy_row + i * ROWS_AT_ONCE;
                const uint32_t at = row * 16 * BITS + 16 * (BITS == 8 ? piece ^ (row & 1) : piece);
                const bool ok = exists && i * ROWS_AT_ONCE < rows_left;
                copy_async16(in + at, ok ? from + i * row_step : a.codes, ok ? 16 : 0);
            }
            from += 16 * BITS * share;
            const int scale_bytes = fc * 128 + 32 * t4 < k ? 4 : 0;
#pragma unroll
            for (int i = 0; i < 2 * R; ++i) {
#pragma unroll
                for (int j = 0; j < NS; ++j)
                    copy_async4(in + CODES + ((i * NS + j) * 32 + lane) * 4,
                                reinterpret_cast<const void *>(scales + (scale_bytes ? scale_from[i] + j * part_step : 0) & ~(uintptr_t)3),
                                scale_bytes);
                scale_from[i] += scale_step;
            }
            in += SLOT;
            if (in == ring_end) in = ring;
            fc += share;
            if (fc >= chunks) {
                fc = warp;
                ft += step;
                enter();
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if constexpr (WHOLE) {
        enter();
#pragma unroll 1
        for (int i = 0; i < AHEAD; ++i) copy_next();
    }
#pragma unroll 1
    for (int t = first; t < sched.total; t += step) {
        const MmaTile tile = mma_tile(m, sched, t, FEATS);
        // rows past the tile repeat its last one; their sums are not stored
        const uint16_t *x0 = static_cast<const uint16_t *>(a.x) + (long long)(tile.r0 + min(g, tile.rows - 1)) * a.x_stride + 32 * t4;
        uint32_t high = 0;   // which 16-bit scales are the high half of their word
        if (WHOLE && !wide) {
#pragma unroll
            for (int i = 0; i < 2 * R; ++i)
#pragma unroll
                for (int j = 0; j < NS; ++j) high |= (uint32_t)(expert_scales(tile.e) + scale_offset(tile.f0 + 8 * i + g) + j * part_step >> 1 & 1) << (i * NS + j);
        }
        float acc[R][4] = {};
#pragma unroll 1
        for (int c = warp; c < chunks; c += share) {
            const int col = c * 128 + 32 * t4, left = WHOLE ? 32 : codes_left(a, col);
            uint32_t xs[2][8];   // on their way while the codes are waited for
#pragma unroll
            for (int h = 0; h < 2; ++h) fetch_x<WHOLE>(xs[h], x0 + c * 128 + 16 * h, k - col - 16 * h);
            CodeRun<KIND> q[2 * R];
            if constexpr (WHOLE) {
                asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
                __syncwarp();
                copy_next();   // into the slot that was read in the step before
#pragma unroll
                for (int i = 0; i < 2 * R; ++i) {
                    const int row = 8 * i + g;
                    const uint32_t at = out + row * 16 * BITS;
                    if constexpr (BITS == 2) {
                        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(q[i].w[0]), "=r"(q[i].w[1]) : "r"(at + 8 * t4) : "memory");
                    } else {
#pragma unroll
                        for (int h = 0; h < BITS / 4; ++h)
                            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                         : "=r"(q[i].w[4 * h]), "=r"(q[i].w[4 * h + 1]), "=r"(q[i].w[4 * h + 2]), "=r"(q[i].w[4 * h + 3])
                                         : "r"(at + 16 * (BITS == 8 ? (2 * t4 + h) ^ (row & 1) : t4))
                                         : "memory");
                    }
#pragma unroll
                    for (int j = 0; j < NS; ++j) {
                        const int s = i * NS + j;
                        uint32_t v;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(out + CODES + (s * 32 + lane) * 4) : "memory");
                        q[i].s[j] = wide ? v : high >> s & 1 ? v >> 16 : v & 0xffffu;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 2 * R; ++i) {
                    CodeRow row = code_row(a, tile.e, min(tile.f0 + 8 * i + g, a.n - 1));
                    row.exists = 1;
                    fetch_run<KIND>(a, q[i], row, col);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t *x = xs[h];
                if constexpr (split_pairs<KIND, NS>) {
#pragma unroll
                    for (int j = 0; j < 8; j += 4) {
                        const uint32_t y0 = x[j], y1 = x[j + 1], y2 = x[j + 2], y3 = x[j + 3];
                        x[j] = __byte_perm(y0, y2, 0x5410);
                        x[j + 1] = __byte_perm(y0, y2, 0x7632);
                        x[j + 2] = __byte_perm(y1, y3, 0x5410);
                        x[j + 3] = __byte_perm(y1, y3, 0x7632);
                    }
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    uint32_t o[2][8];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        decode_half_run<KIND, FDT, NS>(a, q[2 * r + i], h, left, o[i]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_m16n8k16<FDT>(acc[r], o[0][2 * j], o[1][2 * j], o[0][2 * j + 1], o[1][2 * j + 1], x[2 * j], x[2 * j + 1]);
                }
            }
            out += SLOT;
            if (out == ring_end) out = ring;
        }
        // the warps' sums of features g, g + 8 and rows 2 t4, 2 t4 + 1, added in warp order
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[(warp * ROWS + 2 * t4 + (j & 1)) * FEATS + 16 * r + g + (j & 2) * 4] = acc[r][j];
        meet();
        for (int i = warp * 32 + lane; i < ROWS * FEATS; i += 32 * share) {
            const int r = i / FEATS, f = tile.f0 + i % FEATS;
            if (r < tile.rows && f < a.feats) {
                float sum = part[i];
                for (int w = 1; w < share; ++w) sum += part[w * ROWS * FEATS + i];
                finish_one<FDT>(a, tile.r0 + r, f, sum, load_bias<FDT>(a, tile.e, f));
            }
        }
        meet();
    }
    if constexpr (WHOLE) asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- launch -------------------------------------------------------------------------------------------------
template <int KIND, int FDT, int R, int NS>
static cudaError_t launch_skinny_rows(const LinearArgs &a, long long row_tiles, int split, const LaunchCfg &cfg, cudaStream_t stream)
{
    static std::atomic<unsigned long long> ready{0};
    LinearMmaArgs m = {};
    m.a = a;
    m.tile_rows = SKINNY_ROWS;
    m.feat_tiles = (a.feats + SKINNY_FEATS * R - 1) / (SKINNY_FEATS * R);
    m.by_feat_tiles = make_fastdiv((unsigned)m.feat_tiles);
    const long long tiles = row_tiles * m.feat_tiles, resident = cfg.sm_count * (NS < 4 ? 3 : 2);
    m.split = split;
    const size_t smem = skinny_bytes(kind_bits(KIND), R, NS) + (a.offsets ? (3 * a.experts + 1) * 4 : 0);
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {   // devices whose shared-memory limit of this kernel is raised
        e = cudaFuncSetAttribute(linear_skinny_kernel<KIND, FDT, R, NS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t c = {};
    const long long ctas = (tiles * m.split + SKINNY_WARPS - 1) / SKINNY_WARPS;
    c.gridDim = dim3((unsigned)(ctas < resident ? ctas : resident));
    c.blockDim = dim3(32 * SKINNY_WARPS);
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = attr;
    c.numAttrs = cfg.pdl ? 1 : 0;
    return cudaLaunchKernelEx(&c, linear_skinny_kernel<KIND, FDT, R, NS>, m);
}

template <int KIND, int FDT> static cudaError_t launch_skinny_one(const LinearArgs &a, const LaunchCfg &cfg, cudaStream_t stream)
{
    const int scales = skinny_regular(a) ? a.run_scales : 4, chunks = (a.k + 127) / 128;
    const long long busy = a.experts < a.rows ? a.experts : a.rows;   // experts with rows, at most
    long long row_tiles = (a.rows + SKINNY_ROWS - 1) / SKINNY_ROWS, expected = row_tiles;
    if (a.offsets) {
        row_tiles += busy;   // at most
        expected = busy + a.rows / 32;
    }
    // 32 features a block (x is fetched half as often) where that leaves three blocks for each CTA and three CTAs fit an SM,
    // which those of 8-bit codes do not; else 16.  Four warps to a block where eight leave each CTA eight blocks (half as
    // many sums to add); fewer where K has fewer chunks.  One row, 14336 x 4096 q4, 16 features and 8 warps (3 rounds) 19 us, 32 and
    // 4 (1 round) 26; one row for each of 8 experts, 32 and 4 (5 rounds) 59 us, 32 and 8 (9 rounds) 69.
    const long long ctas = (long long)cfg.sm_count * (scales < 4 ? 3 : 2);
    const auto blocks = [&](int r) { return expected * ((a.feats + 16 * r - 1) / (16 * r)); };
    const int best_r = scales < 4 && kind_bits(KIND) < 8 && blocks(2) > 2 * ctas ? 2 : 1;
    int split = blocks(best_r) > 7 * ctas ? 4 : 8;
    while (split > 2 && split / 2 >= chunks) split /= 2;
    if (scales == 4) return launch_skinny_rows<KIND, FDT, 1, 4>(a, row_tiles, split, cfg, stream);
    if constexpr (kind_bits(KIND) < 8) {
        if (best_r == 2)
            return scales == 1 ? launch_skinny_rows<KIND, FDT, 2, 1>(a, row_tiles, split, cfg, stream)
                               : launch_skinny_rows<KIND, FDT, 2, 2>(a, row_tiles, split, cfg, stream);
    }
    return scales == 1 ? launch_skinny_rows<KIND, FDT, 1, 1>(a, row_tiles, split, cfg, stream)
                       : launch_skinny_rows<KIND, FDT, 1, 2>(a, row_tiles, split, cfg, stream);
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
