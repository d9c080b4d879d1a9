// What the tensor-core kernels of the products with quantized weights share: the schedule of tiles, and the warps that bring the
// weight to shared memory.
#pragma once

#include <atomic>
#include <type_traits>

#include "linear_kernels.cuh"
#include "sm100.cuh"

namespace qk {

struct LinearMmaArgs {
    LinearArgs a;
    int tile_rows;    // rows of x per tile
    int stages;
    int split;        // CTAs of a cluster that share a tile's contraction
    int feat_tiles;
    FastDiv by_feat_tiles;
    int tmem_columns;
    int kblocks;      // steps of 64 of the contraction
    // Where aligned rows, whole steps and blocks allow it, codes are fetched as tiles, and a thread's scales lie a constant
    // number of bytes apart from one of its group's steps to the next.
    int regular;
    long long scale_step;
};

constexpr int MMA_MAX_STAGES = 8;
constexpr int MMA_SMEM_LIMIT = 451 * 512;   // dynamic, of 227 KiB; the barriers are static

struct MmaTile {
    int e, f0, r0, rows;
};

// Offsets of the tiles of each expert, in shared memory; experts == 1 needs none.
struct MmaSchedule {
    int total;          // tiles of all experts
    int one_rows;       // a.offsets == nullptr
    const int *prefix;  // [experts + 1] tiles of rows before expert e
    const int *lo, *hi;
};

__device__ __forceinline__ MmaTile mma_tile(const LinearMmaArgs &m, const MmaSchedule &s, int t, int feats_per_tile)
{
    MmaTile r;
    const int rt = (int)fastdiv((unsigned)t, m.by_feat_tiles);
    r.f0 = (t - rt * m.feat_tiles) * feats_per_tile;
    if (s.prefix == nullptr) {
        r.e = 0;
        r.r0 = rt * m.tile_rows;
        r.rows = min(m.tile_rows, s.one_rows - r.r0);
        return r;
    }
    int a = 0, b = m.a.experts;   // prefix[a] <= rt < prefix[b]
    while (b - a > 1) {
        const int mid = (a + b) / 2;
        if (s.prefix[mid] <= rt) a = mid;
        else b = mid;
    }
    r.e = a;
    r.r0 = s.lo[a] + (rt - s.prefix[a]) * m.tile_rows;
    r.rows = min(m.tile_rows, s.hi[a] - r.r0);
    return r;
}

// The schedule of all CTAs, from the offsets; `table` has room for 3 experts + 1 ints.  All `threads` of the CTA call it.
__device__ __forceinline__ MmaSchedule mma_schedule(const LinearMmaArgs &m, int *table, int threads)
{
    const LinearArgs &a = m.a;
    MmaSchedule s;
    s.prefix = s.lo = s.hi = nullptr;
    s.one_rows = a.rows;
    if (a.offsets == nullptr) {
        s.total = (a.rows + m.tile_rows - 1) / m.tile_rows * m.feat_tiles;
        return s;
    }
    int *prefix = table, *lo = table + a.experts + 1, *hi = lo + a.experts;
    const int lane = threadIdx.x % 32;
    int descend = 0;
    for (int e = threadIdx.x; e < a.experts; e += threads) {
        int l, h;
        descend |= expert_rows(a, e, l, h);
        lo[e] = l;
        hi[e] = h;
    }
    // Only offsets that descend somewhere can name a row twice.  It goes to the first expert: two would write it in any order,
    // and the tiles would be more than were counted before the launch.
    if (__syncthreads_or(descend)) {
        if (threadIdx.x == 0) {
            int taken = 0;
            for (int e = 0; e < a.experts; ++e) {
                lo[e] = max(lo[e], taken);
                hi[e] = max(hi[e], lo[e]);
                if (hi[e] > lo[e]) taken = hi[e];
            }
        }
        __syncthreads();
    }
    if (threadIdx.x < 32) {   // running sum of the experts' tiles of rows
        int sum = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 32) {
            const int e = e0 + lane;
            int n = e < a.experts ? (hi[e] - lo[e] + m.tile_rows - 1) / m.tile_rows : 0;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int up = __shfl_up_sync(0xffffffffu, n, d);
                if (lane >= d) n += up;
            }
            if (e < a.experts) prefix[e + 1] = sum + n;
            sum += __shfl_sync(0xffffffffu, n, 31);
        }
        if (lane == 0) prefix[0] = 0;
    }
    __syncthreads();
    s.prefix = prefix;
    s.lo = lo;
    s.hi = hi;
    s.total = prefix[a.experts] * m.feat_tiles;
    return s;
}

// ---- weight --------------------------------------------------------------------------------------------------
// A group of 128 threads brings 64 x 64 codes at a time from memory to the layout that the instructions read: a thread
// takes 32 codes of a row, turns them into 16-bit floats and stores them as four 16-byte chunks of a swizzled row of
// 128 bytes.  Rows are weight rows: features forward (the tile is K-major), steps of the contraction backward (MN-major).
// Groups take the steps in turn (counted through all tiles of the CTA), so that one hides the other's latencies: with two
// warps a scheduler a step of 128 x 64 codes took 1700 cycles, whatever was taken out of it.
constexpr int WEIGHT_THREADS = 128, WEIGHT_GROUPS = 4, WEIGHT_SCALES_AHEAD = 4;

// Shared memory of the codes and scales in flight; `scales` of a run, 0: not regular.
__host__ __device__ constexpr int weight_bytes(int kind, int scales, int slots)
{
    return scales == 0 ? WEIGHT_GROUPS * (kind_bits(kind) >= 4 ? StagedRuns<KIND_I8>::AHEAD : StagedRuns<KIND_PACK2>::AHEAD) * WEIGHT_THREADS *
                             (kind_bits(kind) * 4 + 20)
                       : slots * 512 * kind_bits(kind) + WEIGHT_GROUPS * WEIGHT_SCALES_AHEAD * WEIGHT_THREADS * 4 * scales;
}
// Of every kind of code: 8-bit ones take most either way, or 2-bit ones, whose irregular runs are copied a step further ahead.
__host__ __device__ constexpr int weight_bytes_most(int slots)
{
    int most = 0;
    for (const int kind : {KIND_I8, KIND_PACK4, KIND_PACK2})
        for (const int scales : {0, 1, 2}) most = weight_bytes(kind, scales, slots) > most ? weight_bytes(kind, scales, slots) : most;
    return most;
}
// Shared memory beside stages and runs: up to a boundary of 1 KiB, and the table of the most experts.
constexpr int MMA_SMEM_OTHER = 1024 + (3 * QK_LINEAR_MAX_EXPERTS + 1) * 4;

// STRIDE: steps from one of a group's to its next.  SLOTS: tiles of codes in flight to the CTA; a group takes every fourth.
template <int KIND, int FDT, bool BWD, int STRIDE, int SLOTS> struct WeightWarps {
    static constexpr int BITS = kind_bits(KIND), TILE_BYTES = 512 * BITS;
    const LinearMmaArgs &m;
    const MmaSchedule &sched;
    int first, step;       // tiles of the CTA
    int kb0, kb1;          // its steps of the contraction
    int group, offset;     // the group, and its first step
    int id;                // thread of the group
    int feats_per_tile, f_offset;
    uint32_t runs;         // shared memory of codes and scales

    // Waits and hands over the 16 registers of each run: wait(barrier, parity), put(registers), finish_tile().
    template <class Wait, class Put, class Finish, class Full, class Empty>
    __device__ __forceinline__ void run(const Wait &wait, const Put &put, const Finish &finish_tile, const Full &codes_full, const Empty &codes_empty,
                                        const bool &dead)
    {
        if (kb0 >= kb1) {
            for (int t = first; t < sched.total; t += step) finish_tile();
            return;
        }
        const LinearArgs &a = m.a;
        const int steps = kb1 - kb0, r = id / 2, run_col = (id & 1) * 32, lane = threadIdx.x % 32;
        const auto features = [&](const MmaTile &tile) { return tile.f0 + f_offset; };
        // the step whose codes or scales are copied next: tile and step of the contraction
        int it = first, ikb = kb0 + offset;
        const auto wrap = [&] {
            while (ikb >= kb1) {
                ikb -= steps;
                it += step;
            }
        };
        // Tiles of codes come by bulk tensor copies, a run's scales (one or two) by the thread's own asynchronous copies.
        // (All by the threads' own copies, 16 lines an access: 530 us instead of 493 for 4096 x 14336 x 4096.)
        const auto regular = [&](auto ns) {
            constexpr int NS = decltype(ns)::value, AHEAD = WEIGHT_SCALES_AHEAD;
            constexpr uint32_t SCALE_SLOT = NS * WEIGHT_THREADS * 4;
            const uint32_t ring = runs + SLOTS * TILE_BYTES + group * AHEAD * SCALE_SLOT + id * 4, ring_end = ring + AHEAD * SCALE_SLOT;
            const int scale_size = a.param == QK_F32 ? 4 : 2;
            const long long part = (long long)scale_size * a.scale_col;   // from one of a run's scales to the next
            const bool moving = m.scale_step != 0 || NS > 1;
            const auto scale_at = [&](const MmaTile &tile, int kb) -> uintptr_t {   // 0: past the weight
                const int row = BWD ? kb * 64 + r : features(tile) + r, col = BWD ? features(tile) + run_col : kb * 64 + run_col;
                if (row >= a.n || col >= a.k) return 0;
                return reinterpret_cast<uintptr_t>(a.scales) + scale_index(a, code_row(a, tile.e, row), col) * scale_size;
            };
            // where the thread's run of a tile starts: chunks of 16 bytes, swizzled as the tensor map says
            const uint32_t row_at = r * 8 * BITS;
            const uint32_t chunk = run_col * BITS / 128;
            const uint32_t swizzle = BITS == 8 ? (r >> 1) & 3 : 0;
            uint32_t in = ring, out = ring;
            uintptr_t scale = 0;
            const auto enter = [&] {
                wrap();
                if (it < sched.total) scale = scale_at(mma_tile(m, sched, it, feats_per_tile), ikb);
            };
            const auto copy_next = [&] {
                if (it < sched.total) {
#pragma unroll
                    for (int i = 0; i < NS; ++i)
                        copy_async4(in + i * WEIGHT_THREADS * 4,
                                    reinterpret_cast<const void *>((scale ? scale + i * part : reinterpret_cast<uintptr_t>(a.scales)) & ~(uintptr_t)3), scale ? 4 : 0);
                    in += SCALE_SLOT;
                    if (in == ring_end) in = ring;
                    ikb += STRIDE;
                    if (ikb >= kb1) enter();
                    else if (scale) scale += m.scale_step;
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            if (moving) {
                enter();
#pragma unroll 1
                for (int i = 0; i < AHEAD - 1; ++i) copy_next();
            }
            int kb = kb0 + offset, slot = group, slot_phase = 0;
#pragma unroll 1
            for (int t = first; t < sched.total; t += step) {
                uintptr_t at = 0;   // address of the decoded run's scale
                CodeRun<KIND> run;
                if (!moving || a.param != QK_F32) {
                    at = scale_at(mma_tile(m, sched, t, feats_per_tile), moving ? kb : kb0);
                    if (!moving)
                        run.s[0] = !at ? 0u
                                   : a.param == QK_F32 ? __ldg(reinterpret_cast<const uint32_t *>(at))
                                                       : (uint32_t)__ldg(reinterpret_cast<const unsigned short *>(at));
                }
#pragma unroll 1
                for (; kb < kb1; kb += STRIDE) {
                    uint32_t o[16];
                    if (moving) {
                        copy_next();
                        asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
#pragma unroll
                        for (int i = 0; i < NS; ++i) run.s[i] = take_scale(a, out + i * WEIGHT_THREADS * 4, (unsigned)at + (unsigned)(i * part));
                        at += (unsigned)m.scale_step;
                        out += SCALE_SLOT;
                        if (out == ring_end) out = ring;
                    }
                    wait(codes_full(slot), slot_phase);
                    const uint32_t tile_at = runs + slot * TILE_BYTES + row_at;
                    if constexpr (BITS == 2) {
                        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(run.w[0]), "=r"(run.w[1]) : "r"(tile_at + run_col / 4) : "memory");
                    } else {
#pragma unroll
                        for (int i = 0; i < BITS / 4; ++i)
                            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                         : "=r"(run.w[4 * i]), "=r"(run.w[4 * i + 1]), "=r"(run.w[4 * i + 2]), "=r"(run.w[4 * i + 3])
                                         : "r"(tile_at + 16 * ((chunk + i) ^ swizzle))
                                         : "memory");
                    }
                    decode_code_run<KIND, FDT, NS, true>(a, run, 32, o);
                    __syncwarp();
                    if (lane == 0 && !dead) mbar_arrive(codes_empty(slot));
                    slot += WEIGHT_GROUPS;
                    if (slot >= SLOTS) {
                        slot -= SLOTS;
                        slot_phase ^= 1;
                    }
                    put(o);
                }
                kb -= steps;
                finish_tile();
            }
        };
        // Anything else: codes by the thread's own copies too, every size and alignment.
        const auto irregular = [&] {
            constexpr int AHEAD = StagedRuns<KIND>::AHEAD;
            constexpr uint32_t slot_bytes = StagedRuns<KIND>::slot_bytes(WEIGHT_THREADS);
            const uint32_t slots = runs + group * AHEAD * slot_bytes, slots_end = slots + AHEAD * slot_bytes;
            uint32_t in_slot = slots, out_slot = slots;
            MmaTile itile = {};
            CodeRow irow = {};
            const auto enter = [&] {
                wrap();
                if (it >= sched.total) return;
                itile = mma_tile(m, sched, it, feats_per_tile);
                if (!BWD) irow = code_row(a, itile.e, features(itile) + r);
            };
            const auto copy_next = [&] {
                if (it < sched.total) {
                    if (BWD) irow = code_row(a, itile.e, ikb * 64 + r);
                    stage_code_run<KIND>(a, in_slot, id, WEIGHT_THREADS, irow, BWD ? features(itile) + run_col : ikb * 64 + run_col);
                    in_slot += slot_bytes;
                    if (in_slot == slots_end) in_slot = slots;
                    ikb += STRIDE;
                    if (ikb >= kb1) enter();
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            enter();
#pragma unroll 1
            for (int i = 0; i < AHEAD - 1; ++i) copy_next();
            int kb = kb0 + offset;
#pragma unroll 1
            for (int t = first; t < sched.total; t += step) {
                const MmaTile tile = mma_tile(m, sched, t, feats_per_tile);
                CodeRow row = {};
                if (!BWD && a.param != QK_F32) row = code_row(a, tile.e, features(tile) + r);
#pragma unroll 1
                for (; kb < kb1; kb += STRIDE) {
                    copy_next();
                    asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
                    CodeRun<KIND> run;
                    uint32_t o[16];
                    const int col = BWD ? features(tile) + run_col : kb * 64 + run_col;
                    if (BWD && a.param != QK_F32) row = code_row(a, tile.e, kb * 64 + r);
                    const unsigned skip =
                        a.code_align >= 4 ? 0u : 3u & ((unsigned)reinterpret_cast<uintptr_t>(a.codes) + (unsigned)tile.e * (unsigned)a.code_expert +
                                                       (unsigned)(BWD ? kb * 64 + r : features(tile) + r) * (unsigned)a.code_row);
                    take_codes<KIND>(run, out_slot, id, WEIGHT_THREADS, skip);
                    const uint32_t from = out_slot + WEIGHT_THREADS * CodeRun<KIND>::WORDS * 4 + id * 4;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = i * a.run_scales / 4, part = 32 / a.run_scales;
                        unsigned at = 0;
                        if (a.param != QK_F32) at = (unsigned)reinterpret_cast<uintptr_t>(a.scales) + 2u * (unsigned)scale_index(a, row, col + part * j);
                        run.s[i] = take_scale(a, from + j * WEIGHT_THREADS * 4, at);
                    }
                    out_slot += slot_bytes;
                    if (out_slot == slots_end) out_slot = slots;
                    decode_code_run<KIND, FDT, 4, false>(a, run, codes_left(a, col), o);
                    put(o);
                }
                kb -= steps;
                finish_tile();
            }
        };
        if (!m.regular) irregular();
        else if (a.run_scales == 1) regular(std::integral_constant<int, 1>{});
        else regular(std::integral_constant<int, 2>{});
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
};

// Whether the weight's steps are regular, and how far apart a group's scales.
inline void mma_steps(LinearMmaArgs &m, bool backward, int stride)
{
    const LinearArgs &a = m.a;
    const long long rows = 64 * stride, size = a.param == QK_F32 ? 4 : 2;
    const unsigned block = backward ? a.bn.div : a.bk.div;
    const long long scale_step = backward ? a.scale_row : a.scale_col;
    const bool one = scale_step == 0;
    // two scales of a run are neighbours in blocks of 16 alone: of 48, one run has both halves in one block
    m.regular = a.code_align == 16 && a.k % 32 == 0 && a.contraction % 64 == 0 && (a.run_scales == 1 || a.bk.div == 16) && (one || rows % block == 0);
    m.scale_step = one ? 0 : rows / block * scale_step * size;
}

// ---- launch -------------------------------------------------------------------------------------------------
template <class Kernel>
static cudaError_t launch_cluster(Kernel *kernel, int cluster, int threads, const CUtensorMap &xmap, const CUtensorMap &wmap, const LinearMmaArgs &m, int grid,
                                  size_t smem, const LaunchCfg &cfg, cudaStream_t stream, std::atomic<unsigned long long> &ready)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {   // devices whose shared-memory limit of this kernel is raised
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MMA_SMEM_LIMIT);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((unsigned)grid);
    c.blockDim = dim3((unsigned)threads);
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cfg.pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    c.attrs = attr;
    c.numAttrs = n;
    return cudaLaunchKernelEx(&c, kernel, xmap, wmap, m);
}

}  // namespace qk
