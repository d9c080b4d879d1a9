// Products with quantized weights on the tensor cores: the weight is dequantized into shared memory on the way.
//
// The product is computed transposed, D^T [features, rows]: a tile has 128 features (256 for a pair of CTAs) as the
// instruction's M and up to 256 rows of x as its N, so that a single row of x costs a tile of 16, not of 128.  Per step of 64
// of the contraction, eight warps load codes and scales into registers (several steps ahead, the only way the
// weight is read), turn them into f16 / bf16 and store them to the swizzled layout the instruction reads; one thread loads
// the tile of x by bulk tensor copy; one thread issues the products; four warps take finished tiles from TMEM through the
// epilogue while the next tile runs in the other half of TMEM.
//   forward:  A [128 features = weight rows][64 columns], contraction contiguous (K-major)
//   backward: A [128 features = weight columns][64 weight rows], features contiguous (MN-major): the codes are
//             stored as they lie in memory and the instruction transposes
// Few tiles: the contraction is split over a cluster of CTAs; each sends the others their share of its sums through
// distributed shared memory and adds what it receives in rank order, so results do not depend on timing.
#pragma once

#include <atomic>
#include <type_traits>

#include "linear_kernels.cuh"
#include "sm100.cuh"

namespace qk {

struct LinearMmaArgs {
    LinearArgs a;
    int tile_rows;    // rows of x per tile: a multiple of 16, at most 256
    int stages;
    int split;        // CTAs of a cluster that share a tile's contraction
    int feat_tiles;
    int tmem_columns;
    int kblocks;      // steps of 64 of the contraction
    // Where aligned rows, whole steps and blocks allow it, codes are fetched as tiles, and a thread's scales lie a constant
    // number of bytes apart from one of its group's steps to the next.
    int regular;
    long long scale_step;
};

constexpr int MMA_GROUPS = 2;          // groups of 8 warps that take the weight's steps in turn
constexpr int MMA_WEIGHT_THREADS = 256;
constexpr int MMA_WEIGHT_FIRST = 224;  // warps 0-3 epilogue, 4 loads x, 5 products, 6 loads codes, then weight
constexpr int MMA_THREADS = MMA_WEIGHT_FIRST + MMA_GROUPS * MMA_WEIGHT_THREADS;
constexpr int MMA_MAX_STAGES = 8;
// Tiles of codes on their way, each one step (128 x 64 codes).
template <int KIND> struct CodeTiles {
    static constexpr int BYTES = 128 * 64 * kind_bits(KIND) / 8;
    static constexpr int SLOTS = kind_bits(KIND) == 8 ? 6 : 8;
    static constexpr int SCALES_AHEAD = 4;   // steps of a group whose scales are in flight
};
constexpr int MMA_MAX_CODE_TILES = 8;
constexpr int A_BYTES = 128 * 64 * 2;
constexpr int MMA_SMEM_LIMIT = 226 * 1024;   // dynamic; the barriers are static

// Shared memory of the codes and scales in flight; `scales` of a run, 0: not regular.
__host__ __device__ inline int mma_run_bytes(int kind, int scales)
{
    const int bits = kind_bits(kind), ahead = bits == 8 ? StagedRuns<KIND_I8>::AHEAD : StagedRuns<KIND_PACK4>::AHEAD;
    if (scales == 0) return MMA_GROUPS * ahead * MMA_WEIGHT_THREADS * (bits * 4 + 16);
    return (bits == 8 ? CodeTiles<KIND_I8>::SLOTS : CodeTiles<KIND_PACK4>::SLOTS) * 1024 * bits +
           MMA_GROUPS * CodeTiles<KIND_I8>::SCALES_AHEAD * MMA_WEIGHT_THREADS * 4 * scales;
}

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
    const int rt = t / m.feat_tiles;
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

// 16 sums of one feature per lane, rows row .. row + 15 of which `valid` exist.
template <int FDT>
__device__ __forceinline__ void mma_store16(const LinearArgs &a, float *v, int row, int valid, int f, float bias, float bias_even, float bias_odd)
{
    using F = typename ElemOf<FDT>::type;
    if (a.pairs) {
        // lanes 2i and 2i + 1 hold neighbouring features: the even one takes both of even rows, the odd one of odd rows
        const int odd = threadIdx.x & 1;
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            const float got = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
            v[j] = (odd ? got : v[j]) + bias_even;
            v[j + 1] = (odd ? v[j + 1] : got) + bias_odd;
        }
        if (f >= a.feats) return;
        const long long r0 = row + odd;
        const int fe = f - odd;
        if (a.pre) {
            F *p = static_cast<F *>(a.pre) + r0 * a.pre_stride + fe;
#pragma unroll
            for (int j = 0; j < 16; j += 2)
                if (j + odd < valid) *reinterpret_cast<uint32_t *>(p + j * a.pre_stride) = h2_pack<FDT>(v[j], v[j + 1]);
        }
        activate_all<16>(a.act, v);
        if (a.residual) {
            const F *p = static_cast<const F *>(a.residual) + r0 * a.residual_stride + fe;
            uint32_t q[8];
#pragma unroll
            for (int j = 0; j < 16; j += 2) q[j / 2] = j + odd < valid ? *reinterpret_cast<const uint32_t *>(p + j * a.residual_stride) : 0u;
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                v[j] += widen_lo<FDT>(q[j / 2]);
                v[j + 1] += widen_hi<FDT>(q[j / 2]);
            }
        }
        F *p = static_cast<F *>(a.out) + r0 * a.out_stride + fe;
#pragma unroll
        for (int j = 0; j < 16; j += 2)
            if (j + odd < valid) *reinterpret_cast<uint32_t *>(p + j * a.out_stride) = h2_pack<FDT>(v[j], v[j + 1]);
    } else {
        if (f >= a.feats) return;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            v[j] += bias;
            if (a.pre && j < valid) static_cast<F *>(a.pre)[(row + j) * a.pre_stride + f] = (F)v[j];
        }
        activate_all<16>(a.act, v);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if (j >= valid) break;
            if (a.residual) v[j] += (float)static_cast<const F *>(a.residual)[(row + j) * a.residual_stride + f];
            static_cast<F *>(a.out)[(row + j) * a.out_stride + f] = (F)v[j];
        }
    }
}

// CG: 1, or 2 for a pair of CTAs that works on one tile of 256 features with 2-CTA instructions.
template <int KIND, int FDT, bool BWD, int CG>
__global__ void __launch_bounds__(MMA_THREADS, 1) linear_mma_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const LinearMmaArgs m)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * MMA_MAX_STAGES + 2 * MMA_MAX_CODE_TILES + 5];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const LinearArgs &a = m.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int b_rows = m.tile_rows / CG;                        // rows of x this CTA loads
    const uint32_t b_bytes = (uint32_t)b_rows * 128u, stage_bytes = A_BYTES + b_bytes;
    const uint32_t runs = base + m.stages * stage_bytes;
    int *table = reinterpret_cast<int *>(smem_raw + (runs - smem_u32(smem_raw)) + mma_run_bytes(KIND, m.regular ? a.run_scales : 0));
    const uint32_t bar0 = smem_u32(bars);
    const auto full = [&](int s) { return bar0 + 8u * s; };
    const auto empty = [&](int s) { return bar0 + 8u * (MMA_MAX_STAGES + s); };
    const auto acc_full = [&](int b) { return bar0 + 8u * (2 * MMA_MAX_STAGES + b); };
    const auto acc_empty = [&](int b) { return bar0 + 8u * (2 * MMA_MAX_STAGES + 2 + b); };
    const uint32_t drained = bar0 + 8u * (2 * MMA_MAX_STAGES + 4);
    const auto codes_full = [&](int s) { return bar0 + 8u * (2 * MMA_MAX_STAGES + 5 + s); };
    const auto codes_empty = [&](int s) { return bar0 + 8u * (2 * MMA_MAX_STAGES + 5 + MMA_MAX_CODE_TILES + s); };
    const uint32_t rank = (CG == 2 || m.split > 1) ? cluster_rank() : 0u;
    const bool leader = CG == 1 || rank == 0;

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < MMA_MAX_STAGES; ++s) {
            mbar_init(full(s), 1 + 8 * CG);   // the tile of x (with its bytes) and the warps of the weight
            mbar_init(empty(s), 1);
        }
        for (int s = 0; s < MMA_MAX_CODE_TILES; ++s) {
            mbar_init(codes_full(s), 1);
            mbar_init(codes_empty(s), 8);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), 4 * CG);
        }
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) tmem_alloc<CG>(smem_u32(&tmem_slot), m.tmem_columns);
    pdl_entry();

    MmaSchedule sched;
    sched.prefix = nullptr;
    sched.one_rows = a.rows;
    if (a.offsets != nullptr) {
        int *prefix = table, *lo = table + a.experts + 1, *hi = lo + a.experts;
        for (int e = threadIdx.x; e < a.experts; e += MMA_THREADS) {
            int l, h;
            expert_rows(a, e, l, h);
            lo[e] = l;
            hi[e] = h;
        }
        __syncthreads();
        if (warp == 0) {   // running sum of the experts' tiles of rows
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
        sched.prefix = prefix;
        sched.lo = lo;
        sched.hi = hi;
        sched.total = prefix[a.experts] * m.feat_tiles;
    } else {
        sched.total = (a.rows + m.tile_rows - 1) / m.tile_rows * m.feat_tiles;
    }
    tc_fence_before();
    __syncthreads();
    if (CG == 2 || m.split > 1) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    // Every wait is bounded: a thread that gives up says so to the others of its CTA and to the host, and from then on
    // waits for nothing and starts nothing.
    bool dead = false;
    const auto wait = [&](uint32_t bar, uint32_t parity) {
        if (!dead && !mbar_wait(bar, parity, &gave_up)) {
            dead = true;
            *(volatile int *)&gave_up = 1;
            atomicExch(a.error_flag, 1);
        }
    };

    const int members = CG * m.split;
    const int first = blockIdx.x / members, step = gridDim.x / members;
    const int kb0 = CG == 1 ? (int)((long long)m.kblocks * rank / m.split) : 0;
    const int kb1 = CG == 1 ? (int)((long long)m.kblocks * (rank + 1) / m.split) : m.kblocks;
    constexpr int TILE_FEATS = 128 * CG;
    const int stages = m.stages;
    int stage = 0, phase = 0;
    const auto next_stage = [&](int by = 1) {
        stage += by;
        if (stage >= stages) {
            stage -= stages;
            phase ^= 1;
        }
    };
    // With a split contraction the CTAs of a cluster meet twice per tile: all sums are ready (the stages are free and
    // take the exchange), all shares have arrived; then the CTA's own warps meet before the stages are filled again.
    const auto meet = [&] {
        __syncwarp();
        cluster_sync();
    };
    const auto meet_cta = [&] { asm volatile("bar.sync 1, %0;" ::"n"(MMA_THREADS) : "memory"); };

    if (warp == 4) {
        // ---- tile of x ----------------------------------------------------------------------------------
        int started = 0;
        for (int t = first; t < sched.total; t += step) {
            const MmaTile tile = mma_tile(m, sched, t, TILE_FEATS);
            if (lane == 0) {
                for (int kb = kb0; kb < kb1; ++kb) {
                    wait(empty(stage), phase ^ 1);
                    if (dead) break;
                    const uint32_t dst = base + stage * stage_bytes + A_BYTES;
                    if (CG == 1) {
                        mbar_expect_tx(full(stage), b_bytes);
                        tma_load_2d(dst, &xmap, kb * 64, tile.r0, full(stage));
                    } else {
                        if (leader) mbar_expect_tx(full(stage), 2 * b_bytes);
                        tma_load_2d_pair(dst, &xmap, kb * 64, tile.r0 + (int)rank * b_rows, full(stage));
                    }
                    ++started;
                    next_stage();
                }
            }
            if (m.split > 1) {
                meet();
                meet();
                meet_cta();
            }
        }
        if (dead && leader) {   // copies in flight still write to this CTA's memory: wait for them, again within a limit
            for (int i = min(started, m.stages); i > 0; --i) {
                stage = stage == 0 ? m.stages - 1 : stage - 1;
                if (stage == m.stages - 1) phase ^= 1;
                mbar_wait(full(stage), phase, nullptr);
            }
        }
    } else if (warp == 5) {
        // ---- products -----------------------------------------------------------------------------------
        const uint32_t idesc = instr_desc(FDT == QK_BF16, BWD, 128 * CG, m.tile_rows);
        int buf = 0, buf_phase = 0;
        for (int t = first; t < sched.total; t += step) {
            if (leader && kb0 < kb1) {
                wait(acc_empty(buf), buf_phase ^ 1);
                tc_fence_after();
                const uint32_t d = tmem + buf * m.tile_rows;
#pragma unroll 1
                for (int kb = kb0; kb < kb1; ++kb) {
                    wait(full(stage), phase);
                    dead = __any_sync(0xffffffffu, dead);
                    if (dead) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t sa = base + stage * stage_bytes;
                        // K-major: 16 steps are 32 bytes of a swizzled row.  MN-major: two groups of 8 rows of 128 bytes.
                        const uint64_t da = BWD ? smem_desc(sa, 8192, 1024) : smem_desc(sa, 16, 1024), db = smem_desc(sa + A_BYTES, 16, 1024);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            mma_f16<CG>(d, da + i * (BWD ? 2048 / 16 : 32 / 16), db + i * (32 / 16), idesc, kb > kb0 || i > 0);
                        mma_commit<CG>(empty(stage));
                        if (kb == kb1 - 1) mma_commit<CG>(acc_full(buf));
                    }
                    __syncwarp();
                    next_stage();
                }
                buf ^= 1;
                if (buf == 0) buf_phase ^= 1;
            }
            if (m.split > 1) {
                meet();
                meet();
                meet_cta();
            }
        }
        if (leader) {   // nothing may be in flight to TMEM when it is freed
            if (elect_one()) mma_commit<CG>(drained);
            __syncwarp();
            mbar_wait(drained, 0, nullptr);
        }
        __syncwarp();
    } else if (warp == 6) {
        // ---- tiles of codes -------------------------------------------------------------------------------
        constexpr int SLOTS = CodeTiles<KIND>::SLOTS, BITS = kind_bits(KIND);
        int slot = 0, slot_phase = 0, started = 0;
        for (int t = first; t < sched.total; t += step) {
            const MmaTile tile = mma_tile(m, sched, t, TILE_FEATS);
            const int f = tile.f0 + (CG == 2 ? (int)rank * 128 : 0);
            if (lane == 0 && m.regular) {
#pragma unroll 1
                for (int kb = kb0; kb < kb1; ++kb) {
                    wait(codes_empty(slot), slot_phase ^ 1);
                    if (dead) break;
                    mbar_expect_tx(codes_full(slot), CodeTiles<KIND>::BYTES);
                    tma_load_3d(runs + slot * CodeTiles<KIND>::BYTES, &wmap, (BWD ? f : kb * 64) * BITS / 8, BWD ? kb * 64 : f, tile.e, codes_full(slot));
                    ++started;
                    if (++slot == SLOTS) {
                        slot = 0;
                        slot_phase ^= 1;
                    }
                }
            }
            if (m.split > 1) {
                meet();
                meet();
                meet_cta();
            }
        }
        if (dead) {
            for (int i = min(started, SLOTS); i > 0; --i) {
                slot = slot == 0 ? SLOTS - 1 : slot - 1;
                if (slot == SLOTS - 1) slot_phase ^= 1;
                mbar_wait(codes_full(slot), slot_phase, nullptr);
            }
        }
        __syncwarp();
    } else if (warp >= 7) {
        // ---- weight -------------------------------------------------------------------------------------
        // Steps are numbered through all tiles of the CTA; group g takes those that are g modulo the number of groups.  (One
        // group of 8 warps: 1700 cycles a step, the latency of its instructions; they need more warps to hide in.)
        // A thread's 32 codes of a step: 8 neighbouring lanes store to 8 different 16-byte columns of the swizzle.
        const int group = (threadIdx.x - MMA_WEIGHT_FIRST) / MMA_WEIGHT_THREADS, id = (threadIdx.x - MMA_WEIGHT_FIRST) % MMA_WEIGHT_THREADS;
        const int half = BWD ? id / 128 : 0, r = BWD ? (id / 2) % 64 : id / 2, c = (id & 1) * 4;
        const uint32_t mine = BWD ? half * 8192 + r * 128 : r * 128;
        const uint32_t places = 16u * ((unsigned)c ^ (r & 7));   // of the first chunk; the others: exclusive or with 16 j
        const int steps = kb1 - kb0, run_col = half * 64 + (id & 1) * 32;
        const auto features = [&](const MmaTile &tile) { return tile.f0 + (CG == 2 ? (int)rank * 128 : 0); };
        const auto put = [&](const uint32_t *o) {
            wait(empty(stage), phase ^ 1);
            const uint32_t dst = base + stage * stage_bytes + mine + places;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst ^ (uint32_t)(16 * j)), "r"(o[4 * j]), "r"(o[4 * j + 1]),
                             "r"(o[4 * j + 2]), "r"(o[4 * j + 3])
                             : "memory");
            fence_async_shared();
            __syncwarp();
            if (lane == 0 && !dead) {
                if (CG == 1) mbar_arrive(full(stage));
                else mbar_arrive_cluster(full(stage), 0);
            }
            next_stage(MMA_GROUPS);
        };
        const auto finish_tile = [&] {
            if (m.split > 1) {
                meet();
                meet();
                meet_cta();
            }
        };
        // the step whose codes are copied next: tile and step of the contraction
        int it = first, ikb = kb0 + group;
        const auto wrap = [&] {
            while (ikb >= kb1) {
                ikb -= steps;
                it += step;
            }
        };
        // Tiles of codes come by bulk tensor copies, a run's scales (one or two) by the thread's own asynchronous copies.
        // (All by the threads' own copies: 16 rows a warp are 16 lines an access, 530 us instead of TODO.)
        const auto regular = [&](auto ns) {
            constexpr int NS = decltype(ns)::value, AHEAD = CodeTiles<KIND>::SCALES_AHEAD, SLOTS = CodeTiles<KIND>::SLOTS, BITS = kind_bits(KIND);
            constexpr uint32_t SCALE_SLOT = NS * MMA_WEIGHT_THREADS * 4;
            const uint32_t ring = runs + SLOTS * CodeTiles<KIND>::BYTES + group * AHEAD * SCALE_SLOT + id * 4, ring_end = ring + AHEAD * SCALE_SLOT;
            const int scale_size = a.param == QK_F32 ? 4 : 2;
            const long long part = (long long)scale_size * a.scale_col;   // from one of a run's scales to the next
            const bool moving = m.scale_step != 0 || NS > 1;
            const auto scale_at = [&](const MmaTile &tile, int kb) -> uintptr_t {   // 0: past the weight
                const int row = BWD ? kb * 64 + r : features(tile) + r, col = BWD ? features(tile) + run_col : kb * 64 + run_col;
                if (row >= a.n || col >= a.k) return 0;
                return reinterpret_cast<uintptr_t>(a.scales) + scale_index(a, code_row(a, tile.e, row), col) * scale_size;
            };
            // where the thread's run of a tile starts: chunks of 16 bytes, swizzled as the tensor map says
            const uint32_t row_at = BWD ? r * 16 * BITS : r * 8 * BITS;
            const uint32_t chunk = (BWD ? half * 64 + (id & 1) * 32 : (id & 1) * 32) * BITS / 128;
            const uint32_t swizzle = BITS != 8 ? 0 : BWD ? r & 7 : (r >> 1) & 3;
            uint32_t in = ring, out = ring;
            uintptr_t scale = 0;
            const auto enter = [&] {
                wrap();
                if (it < sched.total) scale = scale_at(mma_tile(m, sched, it, TILE_FEATS), ikb);
            };
            const auto copy_next = [&] {
                if (it < sched.total) {
#pragma unroll
                    for (int i = 0; i < NS; ++i)
                        copy_async4(in + i * MMA_WEIGHT_THREADS * 4, reinterpret_cast<const void *>(scale ? (scale + i * part) & ~(uintptr_t)3 : reinterpret_cast<uintptr_t>(a.codes) & ~(uintptr_t)3),
                                    scale ? 4 : 0);
                    in += SCALE_SLOT;
                    if (in == ring_end) in = ring;
                    ikb += MMA_GROUPS;
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
            int kb = kb0 + group, slot = group, slot_phase = 0;
            next_stage(group);
#pragma unroll 1
            for (int t = first; t < sched.total; t += step) {
                uintptr_t at = 0;   // address of the decoded run's scale
                CodeRun<KIND> run;
                if (!moving || a.param != QK_F32) {
                    at = scale_at(mma_tile(m, sched, t, TILE_FEATS), moving ? kb : kb0);
                    if (!moving) run.s[0] = !at ? 0u : a.param == QK_F32 ? __ldg(reinterpret_cast<const uint32_t *>(at)) : (uint32_t)__ldg(reinterpret_cast<const unsigned short *>(at));
                }
#pragma unroll 1
                for (; kb < kb1; kb += MMA_GROUPS) {
                    uint32_t o[16];
                    if (moving) {
                        copy_next();
                        asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
#pragma unroll
                        for (int i = 0; i < NS; ++i) run.s[i] = take_scale(a, out + i * MMA_WEIGHT_THREADS * 4, (unsigned)at + (unsigned)(i * part));
                        at += (unsigned)m.scale_step;
                        out += SCALE_SLOT;
                        if (out == ring_end) out = ring;
                    }
                    wait(codes_full(slot), slot_phase);
                    const uint32_t tile_at = runs + slot * CodeTiles<KIND>::BYTES + row_at;
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
                    slot += MMA_GROUPS;
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
        const auto irregular = [&] {
            constexpr int AHEAD = StagedRuns<KIND>::AHEAD;
            constexpr uint32_t slot_bytes = StagedRuns<KIND>::slot_bytes(MMA_WEIGHT_THREADS);
            const uint32_t slots = runs + group * AHEAD * slot_bytes, slots_end = slots + AHEAD * slot_bytes;
            uint32_t in_slot = slots, out_slot = slots;
            MmaTile itile = {};
            const auto enter = [&] {
                wrap();
                if (it < sched.total) itile = mma_tile(m, sched, it, TILE_FEATS);
            };
            const auto copy_next = [&] {
                if (it < sched.total) {
                    const CodeRow row = code_row(a, itile.e, BWD ? ikb * 64 + r : features(itile) + r);
                    stage_code_run<KIND>(a, in_slot, id, MMA_WEIGHT_THREADS, row, BWD ? features(itile) + run_col : ikb * 64 + run_col);
                    in_slot += slot_bytes;
                    if (in_slot == slots_end) in_slot = slots;
                    ikb += MMA_GROUPS;
                    if (ikb >= kb1) enter();
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            enter();
#pragma unroll 1
            for (int i = 0; i < AHEAD - 1; ++i) copy_next();
            int kb = kb0 + group;
            next_stage(group);
#pragma unroll 1
            for (int t = first; t < sched.total; t += step) {
                const MmaTile tile = mma_tile(m, sched, t, TILE_FEATS);
#pragma unroll 1
                for (; kb < kb1; kb += MMA_GROUPS) {
                    copy_next();
                    asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
                    CodeRun<KIND> run;
                    uint32_t o[16];
                    const int col = BWD ? features(tile) + run_col : kb * 64 + run_col;
                    const CodeRow row = code_row(a, tile.e, BWD ? kb * 64 + r : features(tile) + r);
                    take_codes<KIND>(run, out_slot, id, MMA_WEIGHT_THREADS);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        run.s[i] = take_scale(a, out_slot + MMA_WEIGHT_THREADS * CodeRun<KIND>::WORDS * 4 + (i * MMA_WEIGHT_THREADS + id) * 4,
                                              (unsigned)reinterpret_cast<uintptr_t>(a.scales) + 2u * (unsigned)scale_index(a, row, col + 8 * i));
                    out_slot += slot_bytes;
                    if (out_slot == slots_end) out_slot = slots;
                    decode_code_run<KIND, FDT, 4, false>(a, run, codes_left(a, col), o);
                    put(o);
                }
                kb -= steps;
                finish_tile();
            }
        };
        if (kb0 < kb1) {
            if (!m.regular) irregular();
            else if (a.run_scales == 1) regular(std::integral_constant<int, 1>{});
            else regular(std::integral_constant<int, 2>{});
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
            for (int t = first; t < sched.total; t += step) finish_tile();
        }
    } else {
        // ---- epilogue -----------------------------------------------------------------------------------
        int buf = 0, buf_phase = 0;
        for (int t = first; t < sched.total; t += step) {
            const MmaTile tile = mma_tile(m, sched, t, TILE_FEATS);
            const int f = tile.f0 + (CG == 2 ? (int)rank * 128 : 0) + (int)threadIdx.x;
            const float bias = load_bias<FDT>(a, tile.e, f);
            const float bias_even = __shfl_sync(0xffffffffu, bias, lane & ~1), bias_odd = __shfl_sync(0xffffffffu, bias, lane | 1);
            const uint32_t from = tmem + ((uint32_t)warp << 21) + buf * m.tile_rows;   // lane 32 * warp
            const bool sums = kb0 < kb1;
            if (sums) {
                wait(acc_full(buf), buf_phase);
                dead = __any_sync(0xffffffffu, dead);
                tc_fence_after();
            }
            if (m.split == 1) {
                for (int r = 0; r < tile.rows; r += 16) {
                    float v[16];
                    if (sums) {
                        tmem_load16(from + r, v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = 0.0f;
                    }
                    if (!dead) mma_store16<FDT>(a, v, tile.r0 + r, tile.rows - r, f, bias, bias_even, bias_odd);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0 && sums && !dead) {
                    if (CG == 1) mbar_arrive(acc_empty(buf));
                    else mbar_arrive_cluster(acc_empty(buf), 0);
                }
            } else {
                // rows of the tile in shares of `share`; share i is finished by CTA i
                const int share = m.tile_rows / m.split;
                meet();
                for (int r = 0; r < m.tile_rows; r += 16) {
                    float v[16];
                    if (sums) {
                        tmem_load16(from + r, v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = 0.0f;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int owner = (r + i) / share, at = (r + i) - owner * share;
                        if (r + i < tile.rows) st_cluster_f32(cluster_map(base + ((rank * share + at) * 128 + threadIdx.x) * 4, owner), v[i]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0 && sums && !dead) mbar_arrive(acc_empty(buf));
                meet();
                const float *got = reinterpret_cast<const float *>(smem_raw + (base - smem_u32(smem_raw)));
                const int r0 = (int)rank * share;
                for (int r = 0; r < share && r0 + r < tile.rows; r += 16) {
                    float v[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        v[i] = 0.0f;
                        if (r + i < share && r0 + r + i < tile.rows)
                            for (int s = 0; s < m.split; ++s) v[i] += got[(s * share + r + i) * 128 + threadIdx.x];
                    }
                    if (!dead) mma_store16<FDT>(a, v, tile.r0 + r0 + r, min(share - r, tile.rows - r0 - r), f, bias, bias_even, bias_odd);
                }
                fence_async_shared();   // what was read here is written by bulk copies next
                meet_cta();
            }
            if (sums) {
                buf ^= 1;
                if (buf == 0) buf_phase ^= 1;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (CG == 2 || m.split > 1) cluster_sync();   // a CTA's memory stays until the others have stopped using it
    if (warp == 5) {
        tc_fence_after();
        tmem_free<CG>(tmem, m.tmem_columns);
    }
}

// Whether the weight's steps are regular, and how far apart its scales.
inline void mma_steps(LinearMmaArgs &m, bool backward)
{
    const LinearArgs &a = m.a;
    const long long rows = 64 * MMA_GROUPS, size = a.param == QK_F32 ? 4 : 2;
    const unsigned block = backward ? a.bn.div : a.bk.div;
    const long long scale_step = backward ? a.scale_row : a.scale_col;
    const bool one = scale_step == 0;
    m.regular = a.code_align == 16 && a.k % 32 == 0 && a.contraction % 64 == 0 && a.run_scales <= 2 && (one || rows % block == 0);
    m.scale_step = one ? 0 : rows / block * scale_step * size;
}

// Tile shape of the codes: {bytes, rows} and the swizzle that the kernel undoes.
inline CUtensorMapSwizzle mma_code_box(bool backward, int bits, cuuint32_t *box)
{
    box[0] = (backward ? 128 : 64) * bits / 8;
    box[1] = backward ? 64 : 128;
    box[2] = 1;
    return bits != 8 ? CU_TENSOR_MAP_SWIZZLE_NONE : backward ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
}

// ---- launch -------------------------------------------------------------------------------------------------
template <int KIND, int FDT, bool BWD, int CG>
static cudaError_t launch_mma_one(const CUtensorMap &xmap, const CUtensorMap &wmap, const LinearMmaArgs &m, int grid, size_t smem, const LaunchCfg &cfg, cudaStream_t stream)
{
    static std::atomic<unsigned long long> ready{0};   // devices whose shared-memory limit of this kernel is raised
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(linear_mma_kernel<KIND, FDT, BWD, CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, MMA_SMEM_LIMIT);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((unsigned)grid);
    c.blockDim = dim3(MMA_THREADS);
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cfg.pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (CG * m.split > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = CG * m.split;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    c.attrs = attr;
    c.numAttrs = n;
    return cudaLaunchKernelEx(&c, linear_mma_kernel<KIND, FDT, BWD, CG>, xmap, wmap, m);
}

template <int FDT, bool BWD, int CG>
static cudaError_t launch_mma_kind(int kind, const CUtensorMap &xmap, const CUtensorMap &wmap, const LinearMmaArgs &m, int grid, size_t smem, const LaunchCfg &cfg,
                                   cudaStream_t stream)
{
    switch (kind) {
    case KIND_PACK8:   // bytes either way
    case KIND_I8: return launch_mma_one<KIND_I8, FDT, BWD, CG>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_PACK4: return launch_mma_one<KIND_PACK4, FDT, BWD, CG>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_PACK2: return launch_mma_one<KIND_PACK2, FDT, BWD, CG>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_E2M1: return launch_mma_one<KIND_E2M1, FDT, BWD, CG>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_E4M3: return launch_mma_one<KIND_E4M3, FDT, BWD, CG>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_E5M2: return launch_mma_one<KIND_E5M2, FDT, BWD, CG>(xmap, wmap, m, grid, smem, cfg, stream);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace qk
