// Which kernel a product with a quantized weight takes, and its launch.
#include "host_checks.cuh"
#include "linear_backward.cuh"
#include "linear_narrow.cuh"
#include "linear_skinny.cuh"
#include "linear_wide.cuh"

namespace qk {

#define QK_DECLARE(NAME) cudaError_t NAME(int, const CUtensorMap &, const CUtensorMap &, const LinearMmaArgs &, int, size_t, const LaunchCfg &, cudaStream_t)
QK_DECLARE(launch_narrow_forward_f16);
QK_DECLARE(launch_narrow_forward_bf16);
QK_DECLARE(launch_narrow_backward_f16);
QK_DECLARE(launch_narrow_backward_bf16);
QK_DECLARE(launch_wide_forward_f16);
QK_DECLARE(launch_wide_forward_bf16);
QK_DECLARE(launch_wide_backward_f16);
QK_DECLARE(launch_wide_backward_bf16);
#undef QK_DECLARE
cudaError_t launch_skinny_f16(int, const LinearArgs &, const LaunchCfg &, cudaStream_t);
cudaError_t launch_skinny_bf16(int, const LinearArgs &, const LaunchCfg &, cudaStream_t);

bool product_needs_aligned_rows(long long rows, const void *x, long long stride)
{
    return reinterpret_cast<uintptr_t>(x) % 16 != 0 || (rows > 1 && stride % 8 != 0);
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                 const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled()
{
    static std::atomic<void *> found{nullptr};
    void *p = found.load(std::memory_order_acquire);
    if (!p) {
        cudaDriverEntryPointQueryResult how;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &how) != cudaSuccess ||
            how != cudaDriverEntryPointSuccess)
            return nullptr;
        found.store(p, std::memory_order_release);
    }
    return reinterpret_cast<EncodeTiled>(p);
}

static int round_up(int v, int to) { return (v + to - 1) / to * to; }

// Clusters of 1, 2, 4 or 8 CTAs that run at once with a CTA per SM.  One of 4 or 8 has to lie in one group of SMs: of the 148 SMs
// 132 and 120 take part (cudaOccupancyMaxActiveClusters), and a 16th cluster of 8 waits for another to end: 16 rows of
// 2048 x 4096, 16 tiles, 24.0 us on clusters of 8, 16.5 on clusters of 4; 34 tiles, 30.2 on clusters of 4, 23.5 on those of 2.
static int resident_clusters(int members, const LaunchCfg &cfg)
{
    return members <= 2 ? cfg.sm_count / members : members == 4 ? cfg.sm_count * 33 / 148 : cfg.sm_count * 15 / 148;
}

static cudaError_t launch_mma(int fdt, int kind, bool backward, const LinearArgs &a, const LaunchCfg &cfg, cudaStream_t stream)
{
    LinearMmaArgs m = {};
    m.a = a;
    const bool grouped = a.offsets != nullptr;
    const int average = a.rows / a.experts;
    m.kblocks = (a.contraction + 63) / 64;
    m.feat_tiles = (a.feats + 127) / 128;
    m.by_feat_tiles = make_fastdiv((unsigned)m.feat_tiles);
    const long long partial = !grouped ? 0 : a.experts < a.rows ? a.experts : a.rows;   // tiles of rows that experts may add
    const auto tiles_of = [&](int tile_rows) { return ((a.rows - 1) / tile_rows + 1 + partial) * m.feat_tiles; };
    if (!grouped) m.tile_rows = round_up((a.rows - 1) / ((a.rows + 255) / 256) + 1, 16);
    else m.tile_rows = average >= 128 ? 256 : round_up(2 * average + 1, 16);
    long long tiles = tiles_of(m.tile_rows);
    m.split = 1;
    while (m.split < 8 && tiles <= resident_clusters(m.split * 2, cfg) && m.kblocks / (m.split * 2) >= 4) m.split *= 2;
    // Pairs of CTAs from 160 rows (of an expert, on average): 8 experts 14336 x 4096 q4 with 128 and 159 rows on the other kernel
    // 245 and 279 us, with 160 and 192 on pairs 299 and 308; one 4096 x 4096 with 159 rows 31, with 160 on pairs
    // 28.  Pairs store a row's features from one lane, which rows that start on no 16 bytes would turn into single elements all
    // over memory.
    // Pairs do not split the contraction, so few tiles of a long one are left to the other kernel: a step of it takes twice as
    // long (0.7 to 0.85 us, of a pair 0.30 to 0.37), and the exchange of a split sum as long as some 64.  us of the other
    // kernel and of pairs, a call at a time: 1024 x 14336 with 160 rows 39 and 76, 512 rows 77 and 92, 1024 rows 63 and 94,
    // 2048 rows 100 and 98; 4096 x 14336 with 160 rows 53 and 78, 384 rows 92 and 94, 768 rows 133 and 98; 512 x 4096 with
    // 512 rows 35 and 37, 1024 x 4096 with 512 rows 55 and 37, 4096 x 4096 with 256 rows 41 and 31.
    const long long tiles_wide = tiles_of(WIDE_ROWS);
    const auto rounds = [&](long long count, int members) {
        const int at_once = resident_clusters(members, cfg);
        return (count + at_once - 1) / at_once;
    };
    const long long steps = rounds(tiles, m.split) * ((m.kblocks + m.split - 1) / m.split), steps_wide = rounds(tiles_wide, 2) * m.kblocks;
    const bool wide = average >= 160 && m.kblocks > 0 && a.wide && steps_wide <= 2 * steps + 64;
    if (wide) {
        m.tile_rows = WIDE_ROWS;
        m.split = 1;
        tiles = tiles_wide;
    }
    mma_steps(m, backward, wide ? WEIGHT_GROUPS : 2);
    const int stage_bytes = wide ? WIDE_STAGE : A_BYTES + m.tile_rows * 128, table = grouped ? (3 * a.experts + 1) * 4 : 0;
    const int runs = weight_bytes(kind, m.regular ? a.run_scales : 0, wide ? WIDE_SLOTS : NARROW_SLOTS);
    m.stages = (MMA_SMEM_LIMIT - 1024 - table - runs) / stage_bytes;
    if (m.stages > MMA_MAX_STAGES) m.stages = MMA_MAX_STAGES;
    if (wide) m.stages = WIDE_STAGES;
    m.tmem_columns = 32;
    while (m.tmem_columns < 2 * m.tile_rows) m.tmem_columns *= 2;
    const int members = wide ? 2 : m.split;
    const long long clusters = cfg.sm_count / members;
    const int grid = (int)(tiles < clusters ? tiles : clusters) * members;
    const size_t smem = 1024 + (size_t)m.stages * stage_bytes + runs + table;

    CUtensorMap xmap = {}, wmap = {};
    if (m.kblocks > 0) {
        const EncodeTiled encode = encode_tiled();
        if (!encode) return cudaErrorNotSupported;
        const cuuint32_t ones[3] = {1, 1, 1};
        const cuuint64_t dims[2] = {(cuuint64_t)a.contraction, (cuuint64_t)a.rows};
        const cuuint64_t strides[1] = {(cuuint64_t)(a.rows > 1 ? a.x_stride * 2 : round_up(a.contraction, 8) * 2ll)};
        const cuuint32_t box[2] = {64, (cuuint32_t)(wide ? 128 : m.tile_rows)};
        CUresult r = encode(&xmap, fdt == QK_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(a.x), dims, strides,
                            box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return cudaErrorInvalidValue;
        if (m.regular) {
            // tiles of 64 x 64 codes; rows and experts that there is one of may come with any stride: it is not used
            const int bits = kind_bits(kind);
            const long long row_bytes = (long long)a.k * bits / 8;
            const cuuint64_t wdims[3] = {(cuuint64_t)row_bytes, (cuuint64_t)a.n, (cuuint64_t)a.experts};
            const cuuint64_t wstrides[2] = {(cuuint64_t)(a.n > 1 ? a.code_row : (row_bytes + 15) / 16 * 16),
                                            (cuuint64_t)(a.experts > 1 ? a.code_expert : (row_bytes + 15) / 16 * 16)};
            const cuuint32_t wbox[3] = {(cuuint32_t)(64 * bits / 8), 64, 1};
            r = encode(&wmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t *>(a.codes), wdims, wstrides, wbox, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       bits == 8 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
            if (r != CUDA_SUCCESS) return cudaErrorInvalidValue;
        }
    }
    using Launch = cudaError_t (*)(int, const CUtensorMap &, const CUtensorMap &, const LinearMmaArgs &, int, size_t, const LaunchCfg &, cudaStream_t);
    static constexpr Launch launches[2][2][2] = {
        {{launch_narrow_forward_f16, launch_narrow_forward_bf16}, {launch_narrow_backward_f16, launch_narrow_backward_bf16}},
        {{launch_wide_forward_f16, launch_wide_forward_bf16}, {launch_wide_backward_f16, launch_wide_backward_bf16}}};
    return launches[wide][backward][fdt == QK_BF16](kind, xmap, wmap, m, grid, smem, cfg, stream);
}

// A handful of rows (of an expert, on average): 14336 x 4096 q8 with 8 rows 27 us, with 9 on the tiles of the tensor
// cores 34; of each of 8 experts, q4, 105 and 189 us, q8 162 and 207.
static bool handful(bool backward, const LinearArgs &a) { return !backward && a.k > 0 && a.rows <= SKINNY_ROWS * a.experts; }

// Tiles are numbered by 32-bit integers, and a CTA steps past the last one by less than 2^20.
bool product_tiles_fit(bool backward, const LinearArgs &a)
{
    const bool few = handful(backward, a);
    const long long partial = !a.offsets ? 0 : a.experts < a.rows ? a.experts : a.rows;
    return (a.rows / (few ? SKINNY_ROWS : 16) + 1 + partial) * (a.feats / (few ? SKINNY_FEATS : 128) + 1ll) < (1ll << 31) - (1 << 20);
}

cudaError_t launch_linear_product(int fdt, int kind, bool backward, const LinearArgs &a, const LaunchCfg &cfg, cudaStream_t stream)
{
    if (handful(backward, a))
        return fdt == QK_F16 ? launch_skinny_f16(kind, a, cfg, stream) : launch_skinny_bf16(kind, a, cfg, stream);
    return launch_mma(fdt, kind, backward, a, cfg, stream);
}

}  // namespace qk
