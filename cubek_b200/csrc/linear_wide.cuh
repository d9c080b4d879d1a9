// Products with quantized weights for many rows: D [rows, features] with the rows of x as the instruction's M.
//
// A pair of CTAs works on 512 rows x 128 features with 2-CTA instructions (256 x 128 x 16): each CTA loads 256 rows of x and
// dequantizes 64 features, and the pair's instructions read both halves of the weight.  So a dequantized tile serves 512
// rows instead of the 256 that the transposed form for few rows reaches: the arithmetic of the weight, which is what competes with
// the tensor cores here, is halved.  A row's features lie in one lane, so the epilogue stores 32 bytes per thread.
// The second 256 rows of a tile are left out where an expert or the tensor ends before them.
//   forward:  B [64 features = weight rows][64 columns], contraction contiguous (K-major)
//   backward: B [64 features = weight columns][64 weight rows], features contiguous (MN-major)
#pragma once

#include "linear_tiles.cuh"

namespace qk {

constexpr int WIDE_ROWS = 512, WIDE_FEATS = 128;          // tile of a pair
constexpr int WIDE_FIRST = 224;                           // warps 0-3 epilogue, 4 loads x, 5 products, 6 loads codes, then weight
constexpr int WIDE_THREADS = WIDE_FIRST + WEIGHT_GROUPS * WEIGHT_THREADS;
constexpr int WIDE_X_BYTES = 128 * 64 * 2, WIDE_STAGE = 2 * WIDE_X_BYTES + 64 * 64 * 2;
constexpr int WIDE_SLOTS = 8, WIDE_STAGES = 4;   // 160 KiB, and at most 52 of runs and 12 of table
static_assert(WIDE_STAGES * WIDE_STAGE <= MMA_SMEM_LIMIT - MMA_SMEM_OTHER - weight_bytes_most(WIDE_SLOTS), "the stages do not fit");

// 16 sums of neighbouring features f .. f + 15 of one row.
template <int FDT> __device__ __forceinline__ void wide_store16(const LinearArgs &a, float *v, long long row, int f, const float *bias)
{
    using F = typename ElemOf<FDT>::type;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += bias[i];
    const bool whole = f + 16 <= a.feats;
    const auto put = [&](void *base, long long stride) {
        F *p = static_cast<F *>(base) + row * stride + f;
        if (whole) {
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = h2_pack<FDT>(v[2 * i], v[2 * i + 1]);
            if (a.wide == 32) {
                asm volatile("st.global.v8.u32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]),
                             "r"(o[5]), "r"(o[6]), "r"(o[7])
                             : "memory");
            } else {
                reinterpret_cast<uint4 *>(p)[0] = make_uint4(o[0], o[1], o[2], o[3]);
                reinterpret_cast<uint4 *>(p)[1] = make_uint4(o[4], o[5], o[6], o[7]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (f + i < a.feats) p[i] = (F)v[i];
        }
    };
    if (a.pre) put(a.pre, a.pre_stride);
    activate_all<16>(a.act, v);
    if (a.residual) {
        const F *p = static_cast<const F *>(a.residual) + row * a.residual_stride + f;
        if (whole) {
            uint32_t q[8];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 u = reinterpret_cast<const uint4 *>(p)[i];
                q[4 * i] = u.x;
                q[4 * i + 1] = u.y;
                q[4 * i + 2] = u.z;
                q[4 * i + 3] = u.w;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[2 * i] += widen_lo<FDT>(q[i]);
                v[2 * i + 1] += widen_hi<FDT>(q[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (f + i < a.feats) v[i] += (float)p[i];
        }
    }
    put(a.out, a.out_stride);
}

template <int KIND, int FDT, bool BWD>
__global__ void __launch_bounds__(WIDE_THREADS, 1) linear_wide_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                                                                      const LinearMmaArgs m)
{
    constexpr int BITS = kind_bits(KIND), TILE_BYTES = 64 * 64 * BITS / 8;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * WIDE_STAGES + 2 * WIDE_SLOTS + 5];
    __shared__ float bias_tile[2][WIDE_FEATS];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const LinearArgs &a = m.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t runs = base + WIDE_STAGES * WIDE_STAGE;
    int *table = reinterpret_cast<int *>(smem_raw + (runs - smem_u32(smem_raw)) + weight_bytes(KIND, m.regular ? a.run_scales : 0, WIDE_SLOTS));
    const uint32_t bar0 = smem_u32(bars);
    const auto full = [&](int s) { return bar0 + 8u * s; };
    const auto empty = [&](int s) { return bar0 + 8u * (WIDE_STAGES + s); };
    const auto acc_full = [&](int b) { return bar0 + 8u * (2 * WIDE_STAGES + b); };
    const auto acc_empty = [&](int b) { return bar0 + 8u * (2 * WIDE_STAGES + 2 + b); };
    const uint32_t drained = bar0 + 8u * (2 * WIDE_STAGES + 4);
    const auto codes_full = [&](int s) { return bar0 + 8u * (2 * WIDE_STAGES + 5 + s); };
    const auto codes_empty = [&](int s) { return bar0 + 8u * (2 * WIDE_STAGES + 5 + WIDE_SLOTS + s); };
    const int rank = (int)cluster_rank();
    const bool leader = rank == 0;

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < WIDE_STAGES; ++s) {
            mbar_init(full(s), 1 + 2 * WEIGHT_THREADS / 32);   // the tile of x (with its bytes) and a group's warps of both CTAs
            mbar_init(empty(s), 1);
        }
        for (int s = 0; s < WIDE_SLOTS; ++s) {
            mbar_init(codes_full(s), 1);
            mbar_init(codes_empty(s), WEIGHT_THREADS / 32);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), 8);
        }
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) tmem_alloc<2>(smem_u32(&tmem_slot), 512);
    pdl_entry();
    const MmaSchedule sched = mma_schedule(m, table, WIDE_THREADS);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    // Every wait is bounded: a thread that gives up says so to the others of its CTA and to the host, and from then on
    // waits for nothing and starts nothing.  A wait for a whole sum may take longer by its steps (1.5 us each at most, for rows
    // of codes that start on no word, on a GPU of its own).
    bool dead = false;
    const auto wait = [&](uint32_t bar, uint32_t parity, int sum_steps = 0) {
        if (!dead && !mbar_wait(bar, parity, &gave_up, sum_steps)) {
            dead = true;
            *(volatile int *)&gave_up = 1;
            atomicExch(a.error_flag, 1);
        }
    };
    const int first = blockIdx.x / 2, step = gridDim.x / 2, steps = m.kblocks;
    unsigned n = 0;   // steps so far: stage n % 4, and whether it has been used an odd number of times
    const auto stage = [&] { return (int)(n % WIDE_STAGES); };
    const auto phase = [&] { return n / WIDE_STAGES & 1; };

    if (warp == 4) {
        // ---- rows of x ----------------------------------------------------------------------------------
        for (int t = first; t < sched.total; t += step) {
            const MmaTile tile = mma_tile(m, sched, t, WIDE_FEATS);
            if (lane == 0) {
                const int parts = tile.rows > 256 ? 2 : 1, row = tile.r0 + rank * 128;
#pragma unroll 1
                for (int kb = 0; kb < steps; ++kb) {
                    wait(empty(stage()), phase() ^ 1);
                    if (dead) break;
                    const uint32_t dst = base + stage() * WIDE_STAGE;
                    if (leader) mbar_expect_tx(full(stage()), 2 * parts * WIDE_X_BYTES);
                    tma_load_2d_pair(dst, &xmap, kb * 64, row, full(stage()));
                    if (parts > 1) tma_load_2d_pair(dst + WIDE_X_BYTES, &xmap, kb * 64, row + 256, full(stage()));
                    ++n;
                }
            }
        }
        if (dead && leader) {   // copies in flight still write to this pair's memory: wait for them, again within a limit
            for (int i = min((int)n, WIDE_STAGES); i > 0; --i) {
                --n;
                mbar_wait(full(stage()), phase(), nullptr);
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        // ---- products -----------------------------------------------------------------------------------
        const uint32_t idesc = instr_desc(FDT == QK_BF16, false, 256, WIDE_FEATS) | (BWD ? 1u << 16 : 0u);
        const uint64_t dx0 = smem_desc(base, 16, 1024), dw0 = smem_desc(base + 2 * WIDE_X_BYTES, BWD ? 8192 : 16, 1024);
        int buf = 0, buf_phase = 0;
        if (leader) {
            for (int t = first; t < sched.total; t += step) {
                const MmaTile tile = mma_tile(m, sched, t, WIDE_FEATS);
                const bool second = tile.rows > 256;
                wait(acc_empty(buf), buf_phase ^ 1);
                tc_fence_after();
                const uint32_t d = tmem + buf * 256;
                // A step's eight products take the tensor cores 512 cycles, and this loop has to come round in less.
#pragma unroll 1
                for (int kb = 0; kb < steps; ++kb, ++n) {
                    wait(full(stage()), phase());
                    if (__any_sync(0xffffffffu, dead)) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t at = stage() * (WIDE_STAGE / 16);
                        const uint64_t dx = dx0 + at, dw = dw0 + at;
                        mma_f16<2>(d, dx, dw, idesc, kb > 0);
#pragma unroll
                        for (int i = 1; i < 4; ++i) mma_f16<2>(d, dx + i * (32 / 16), dw + i * (BWD ? 2048 / 16 : 32 / 16), idesc, true);
                        if (second) {
                            mma_f16<2>(d + 128, dx + WIDE_X_BYTES / 16, dw, idesc, kb > 0);
#pragma unroll
                            for (int i = 1; i < 4; ++i)
                                mma_f16<2>(d + 128, dx + WIDE_X_BYTES / 16 + i * (32 / 16), dw + i * (BWD ? 2048 / 16 : 32 / 16), idesc, true);
                        }
                        mma_commit<2>(empty(stage()));
                    }
                    __syncwarp();
                }
                if (elect_one()) mma_commit<2>(acc_full(buf));
                __syncwarp();
                buf ^= 1;
                if (buf == 0) buf_phase ^= 1;
            }
            if (elect_one()) mma_commit_own(drained);   // nothing may be in flight to TMEM when it is freed
            __syncwarp();
            mbar_wait(drained, 0, nullptr);
        }
        __syncwarp();
    } else if (warp == 6) {
        // ---- tiles of codes -------------------------------------------------------------------------------
        int slot = 0, slot_phase = 0, started = 0;
        if (lane == 0 && m.regular) {
            for (int t = first; t < sched.total; t += step) {
                const MmaTile tile = mma_tile(m, sched, t, WIDE_FEATS);
                const int f = tile.f0 + rank * 64;
#pragma unroll 1
                for (int kb = 0; kb < steps; ++kb) {
                    wait(codes_empty(slot), slot_phase ^ 1);
                    if (dead) break;
                    mbar_expect_tx(codes_full(slot), TILE_BYTES);
                    tma_load_3d(runs + slot * TILE_BYTES, &wmap, (BWD ? f : kb * 64) * BITS / 8, BWD ? kb * 64 : f, tile.e, codes_full(slot));
                    ++started;
                    if (++slot == WIDE_SLOTS) {
                        slot = 0;
                        slot_phase ^= 1;
                    }
                }
            }
            if (dead) {
                for (int i = min(started, WIDE_SLOTS); i > 0; --i) {
                    slot = slot == 0 ? WIDE_SLOTS - 1 : slot - 1;
                    if (slot == WIDE_SLOTS - 1) slot_phase ^= 1;
                    mbar_wait(codes_full(slot), slot_phase, nullptr);
                }
            }
        }
        __syncwarp();
    } else if (warp >= 7) {
        // ---- weight -------------------------------------------------------------------------------------
        const int group = (threadIdx.x - WIDE_FIRST) / WEIGHT_THREADS, id = (threadIdx.x - WIDE_FIRST) % WEIGHT_THREADS;
        const int r = id / 2;
        const uint32_t place = base + 2 * WIDE_X_BYTES + r * 128 + 16u * ((unsigned)((id & 1) * 4) ^ (r & 7));
        const auto put = [&](const uint32_t *o) {
            wait(empty(stage()), phase() ^ 1);
            const uint32_t dst = place + stage() * WIDE_STAGE;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst ^ (uint32_t)(16 * j)), "r"(o[4 * j]), "r"(o[4 * j + 1]),
                             "r"(o[4 * j + 2]), "r"(o[4 * j + 3])
                             : "memory");
            fence_async_shared();
            __syncwarp();
            if (lane == 0 && !dead) mbar_arrive_cluster(full(stage()), 0);
            n += WEIGHT_GROUPS;
        };
        n = group;
        WeightWarps<KIND, FDT, BWD, WEIGHT_GROUPS, WIDE_SLOTS> w{m, sched, first, step, 0, steps, group, group, id, WIDE_FEATS, rank * 64, runs};
        w.run(wait, put, [] {}, codes_full, codes_empty, dead);
    } else {
        // ---- epilogue -----------------------------------------------------------------------------------
        int buf = 0, buf_phase = 0;
        for (int t = first; t < sched.total; t += step) {
            const MmaTile tile = mma_tile(m, sched, t, WIDE_FEATS);
            bias_tile[buf][threadIdx.x] = load_bias<FDT>(a, tile.e, tile.f0 + (int)threadIdx.x);
            asm volatile("bar.sync 2, 128;" ::: "memory");   // the other buffer's readers have passed here once since
            wait(acc_full(buf), buf_phase, steps);
            dead = __any_sync(0xffffffffu, dead);
            tc_fence_after();
            const uint32_t from = tmem + ((uint32_t)warp << 21) + buf * 256;
#pragma unroll 1
            for (int part = 0; part < 2; ++part) {
                const int at = part * 256 + rank * 128 + (int)threadIdx.x;
                if (part * 256 + rank * 128 + warp * 32 >= tile.rows) break;
#pragma unroll 1
                for (int c = 0; c < WIDE_FEATS; c += 16) {
                    if (tile.f0 + c >= a.feats) break;
                    float v[16];
                    tmem_load16(from + part * 128 + c, v);
                    if (!dead && at < tile.rows) wide_store16<FDT>(a, v, tile.r0 + at, tile.f0 + c, &bias_tile[buf][c]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && !dead) mbar_arrive_cluster(acc_empty(buf), 0);
            buf ^= 1;
            if (buf == 0) buf_phase ^= 1;
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();   // a CTA's memory stays until the other has stopped using it
    if (warp == 5) {
        tc_fence_after();
        tmem_free<2>(tmem, 512);
    }
}

// ---- launch -------------------------------------------------------------------------------------------------
template <int KIND, int FDT, bool BWD>
static cudaError_t launch_wide_one(const CUtensorMap &xmap, const CUtensorMap &wmap, const LinearMmaArgs &m, int grid, size_t smem, const LaunchCfg &cfg,
                                   cudaStream_t stream)
{
    static std::atomic<unsigned long long> ready{0};
    return launch_cluster(linear_wide_kernel<KIND, FDT, BWD>, 2, WIDE_THREADS, xmap, wmap, m, grid, smem, cfg, stream, ready);
}

template <int FDT, bool BWD>
static cudaError_t launch_wide_kind(int kind, const CUtensorMap &xmap, const CUtensorMap &wmap, const LinearMmaArgs &m, int grid, size_t smem,
                                    const LaunchCfg &cfg, cudaStream_t stream)
{
    switch (kind) {
    case KIND_PACK8:   // bytes either way
    case KIND_I8: return launch_wide_one<KIND_I8, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_PACK4: return launch_wide_one<KIND_PACK4, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_PACK2: return launch_wide_one<KIND_PACK2, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_E2M1: return launch_wide_one<KIND_E2M1, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_E4M3: return launch_wide_one<KIND_E4M3, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_E5M2: return launch_wide_one<KIND_E5M2, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace qk
