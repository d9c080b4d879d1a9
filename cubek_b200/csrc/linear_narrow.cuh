// Products with quantized weights for few rows: D^T [features, rows], the features as the instruction's M.
//
// A tile has 128 features and up to 256 rows of x as the instruction's N, so that a single row of x costs a tile of
// 16, not of 128.  Per step of 64 of the contraction, groups of warps turn codes into f16 / bf16 in the swizzled layout
// the instruction reads; one thread loads the tile of x by bulk tensor copy; one thread issues the products; four warps take
// finished tiles from TMEM through the epilogue while the next tile runs in the other half of TMEM.
//   forward:  A [128 features = weight rows][64 columns], contraction contiguous (K-major)
//   backward: A [128 features = weight columns][64 weight rows], features contiguous (MN-major): the codes are
//             stored as they lie in memory and the instruction transposes
// Few tiles: the contraction is split over a cluster of CTAs; each sends the others their share of its sums through
// distributed shared memory and adds what it receives in rank order, so results do not depend on timing.
#pragma once

#include "linear_tiles.cuh"

namespace qk {

constexpr int NARROW_FEATS = 128, NARROW_SLOTS = 12;
constexpr int NARROW_WEIGHT_FIRST = 224;   // warps 0-3 epilogue, 4 loads x, 5 products, 6 loads codes, then weight
constexpr int NARROW_THREADS = NARROW_WEIGHT_FIRST + WEIGHT_GROUPS * WEIGHT_THREADS;
constexpr int A_BYTES = 128 * 64 * 2;
// three stages at least: the exchange of a split contraction needs 512 bytes a row
static_assert(3 * (A_BYTES + 256 * 128) <= MMA_SMEM_LIMIT - MMA_SMEM_OTHER - weight_bytes_most(NARROW_SLOTS), "the stages do not fit");
static_assert(256 * 512 <= 3 * (A_BYTES + 256 * 128) && 16 * 512 <= 3 * (A_BYTES + 16 * 128), "the exchange does not fit");

// 16 sums of one feature per lane, rows row .. row + 15 of which `valid` exist.
template <int FDT>
__device__ __forceinline__ void narrow_store16(const LinearArgs &a, float *v, int row, int valid, int f, float bias, float bias_even, float bias_odd)
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

template <int KIND, int FDT, bool BWD>
__global__ void __launch_bounds__(NARROW_THREADS, 1) linear_narrow_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const LinearMmaArgs m)
{
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * MMA_MAX_STAGES + 2 * NARROW_SLOTS + 5];
    __shared__ uint32_t tmem_slot;
    __shared__ int gave_up;
    const LinearArgs &a = m.a;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t b_bytes = (uint32_t)m.tile_rows * 128u, stage_bytes = A_BYTES + b_bytes;
    const uint32_t runs = base + m.stages * stage_bytes;
    int *table = reinterpret_cast<int *>(smem_raw + (runs - smem_u32(smem_raw)) + weight_bytes(KIND, m.regular ? a.run_scales : 0, NARROW_SLOTS));
    const uint32_t bar0 = smem_u32(bars);
    const auto full = [&](int s) { return bar0 + 8u * s; };
    const auto empty = [&](int s) { return bar0 + 8u * (MMA_MAX_STAGES + s); };
    const auto acc_full = [&](int b) { return bar0 + 8u * (2 * MMA_MAX_STAGES + b); };
    const auto acc_empty = [&](int b) { return bar0 + 8u * (2 * MMA_MAX_STAGES + 2 + b); };
    const uint32_t drained = bar0 + 8u * (2 * MMA_MAX_STAGES + 4);
    const auto codes_full = [&](int s) { return bar0 + 8u * (2 * MMA_MAX_STAGES + 5 + s); };
    const auto codes_empty = [&](int s) { return bar0 + 8u * (2 * MMA_MAX_STAGES + 5 + NARROW_SLOTS + s); };
    const int rank = m.split > 1 ? (int)cluster_rank() : 0;

    if (threadIdx.x == 0) {
        gave_up = 0;
        for (int s = 0; s < MMA_MAX_STAGES; ++s) {
            mbar_init(full(s), 1 + 2 * WEIGHT_THREADS / 32);   // the tile of x (with its bytes) and two groups of the weight
            mbar_init(empty(s), 1);
        }
        for (int s = 0; s < NARROW_SLOTS; ++s) {
            mbar_init(codes_full(s), 1);
            mbar_init(codes_empty(s), WEIGHT_THREADS / 32);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), 4);
        }
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) tmem_alloc<1>(smem_u32(&tmem_slot), m.tmem_columns);
    pdl_entry();

    const MmaSchedule sched = mma_schedule(m, table, NARROW_THREADS);
    tc_fence_before();
    __syncthreads();
    if (m.split > 1) cluster_sync();
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

    const int first = blockIdx.x / m.split, step = gridDim.x / m.split;
    const int kb0 = (int)((long long)m.kblocks * rank / m.split), kb1 = (int)((long long)m.kblocks * (rank + 1) / m.split);
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
    const auto meet_cta = [&] { asm volatile("bar.sync 1, %0;" ::"n"(NARROW_THREADS) : "memory"); };

    if (warp == 4) {
        // ---- tile of x ----------------------------------------------------------------------------------
        int started = 0;
        for (int t = first; t < sched.total; t += step) {
            const MmaTile tile = mma_tile(m, sched, t, NARROW_FEATS);
            if (lane == 0) {
                for (int kb = kb0; kb < kb1; ++kb) {
                    wait(empty(stage), phase ^ 1);
                    if (dead) break;
                    const uint32_t dst = base + stage * stage_bytes + A_BYTES;
                    mbar_expect_tx(full(stage), b_bytes);
                    tma_load_2d(dst, &xmap, kb * 64, tile.r0, full(stage));
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
        if (dead) {   // copies in flight still write to this CTA's memory: wait for them, again within a limit
            for (int i = min(started, m.stages); i > 0; --i) {
                stage = stage == 0 ? m.stages - 1 : stage - 1;
                if (stage == m.stages - 1) phase ^= 1;
                mbar_wait(full(stage), phase, nullptr);
            }
        }
    } else if (warp == 5) {
        // ---- products -----------------------------------------------------------------------------------
        const uint32_t idesc = instr_desc(FDT == QK_BF16, BWD, 128, m.tile_rows), stage_step = stage_bytes / 16;
        // K-major: 16 steps are 32 bytes of a swizzled row.  MN-major: two groups of 8 rows of 128 bytes.
        const uint64_t da0 = BWD ? smem_desc(base, 8192, 1024) : smem_desc(base, 16, 1024), db0 = smem_desc(base + A_BYTES, 16, 1024);
        int buf = 0, buf_phase = 0;
        for (int t = first; t < sched.total; t += step) {
            if (kb0 < kb1) {
                wait(acc_empty(buf), buf_phase ^ 1);
                tc_fence_after();
                const uint32_t d = tmem + buf * m.tile_rows;
                // What a step costs here bounds few rows: descriptors are made once, and a step adds to them.
#pragma unroll 1
                for (int kb = kb0; kb < kb1; ++kb) {
                    wait(full(stage), phase);
                    if (__any_sync(0xffffffffu, dead)) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t at = (uint32_t)stage * stage_step;
                        mma_f16<1>(d, da0 + at, db0 + at, idesc, kb > kb0);
#pragma unroll
                        for (int i = 1; i < 4; ++i) mma_f16<1>(d, da0 + at + i * (BWD ? 2048 / 16 : 32 / 16), db0 + at + i * (32 / 16), idesc, true);
                        mma_commit<1>(empty(stage));
                    }
                    __syncwarp();
                    next_stage();
                }
                if (elect_one()) mma_commit<1>(acc_full(buf));
                __syncwarp();
                buf ^= 1;
                if (buf == 0) buf_phase ^= 1;
            }
            if (m.split > 1) {
                meet();
                meet();
                meet_cta();
            }
        }
        if (elect_one()) mma_commit<1>(drained);   // nothing may be in flight to TMEM when it is freed
        __syncwarp();
        mbar_wait(drained, 0, nullptr);
        __syncwarp();
    } else if (warp == 6) {
        // ---- tiles of codes -------------------------------------------------------------------------------
        // Lane l serves group l of the weight: its half of every other step, its slots.  (One lane for all of them took 1000
        // cycles a step, which the groups waited for.)
        constexpr int BITS = kind_bits(KIND), TILE_BYTES = 512 * BITS;
        int slot = lane, slot_phase = 0, started = 0, kb = kb0 + lane / 2;
        for (int t = first; t < sched.total; t += step) {
            const MmaTile tile = mma_tile(m, sched, t, NARROW_FEATS);
            if (lane < WEIGHT_GROUPS && m.regular && kb0 < kb1) {
                const int f = tile.f0 + (lane & 1) * 64;
#pragma unroll 1
                for (; kb < kb1; kb += 2) {
                    wait(codes_empty(slot), slot_phase ^ 1);
                    if (dead) continue;
                    mbar_expect_tx(codes_full(slot), TILE_BYTES);
                    tma_load_3d(runs + slot * TILE_BYTES, &wmap, (BWD ? f : kb * 64) * BITS / 8, BWD ? kb * 64 : f, tile.e, codes_full(slot));
                    ++started;
                    slot += WEIGHT_GROUPS;
                    if (slot >= NARROW_SLOTS) {
                        slot -= NARROW_SLOTS;
                        slot_phase ^= 1;
                    }
                }
                kb -= kb1 - kb0;
            }
            if (m.split > 1) {
                meet();
                meet();
                meet_cta();
            }
        }
        if (dead) {
            for (int i = min(started, NARROW_SLOTS / WEIGHT_GROUPS); i > 0; --i) {
                slot -= WEIGHT_GROUPS;
                if (slot < 0) {
                    slot += NARROW_SLOTS;
                    slot_phase ^= 1;
                }
                mbar_wait(codes_full(slot), slot_phase, nullptr);
            }
        }
        __syncwarp();
    } else if (warp >= 7) {
        // ---- weight -------------------------------------------------------------------------------------
        // Two groups take the halves of one step, the other two those of the next.
        const int id = (threadIdx.x - NARROW_WEIGHT_FIRST) % WEIGHT_THREADS, group = (threadIdx.x - NARROW_WEIGHT_FIRST) / WEIGHT_THREADS;
        const int r = id / 2;
        const uint32_t place = base + (group & 1) * 8192 + r * 128 + 16u * ((unsigned)((id & 1) * 4) ^ (r & 7));
        const auto put = [&](const uint32_t *o) {
            wait(empty(stage), phase ^ 1);
            const uint32_t dst = place + stage * stage_bytes;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst ^ (uint32_t)(16 * j)), "r"(o[4 * j]), "r"(o[4 * j + 1]),
                             "r"(o[4 * j + 2]), "r"(o[4 * j + 3])
                             : "memory");
            fence_async_shared();
            __syncwarp();
            if (lane == 0 && !dead) mbar_arrive(full(stage));
            next_stage(2);
        };
        const auto finish_tile = [&] {
            if (m.split > 1) {
                meet();
                meet();
                meet_cta();
            }
        };
        next_stage(group / 2);
        WeightWarps<KIND, FDT, BWD, 2, NARROW_SLOTS> w{m, sched, first, step, kb0, kb1, group, group / 2, id, NARROW_FEATS, (group & 1) * 64, runs};
        w.run(wait, put, finish_tile, codes_full, codes_empty, dead);
    } else {
        // ---- epilogue -----------------------------------------------------------------------------------
        int buf = 0, buf_phase = 0;
        for (int t = first; t < sched.total; t += step) {
            const MmaTile tile = mma_tile(m, sched, t, NARROW_FEATS);
            const int f = tile.f0 + (int)threadIdx.x;
            const float bias = load_bias<FDT>(a, tile.e, f);
            const float bias_even = __shfl_sync(0xffffffffu, bias, lane & ~1), bias_odd = __shfl_sync(0xffffffffu, bias, lane | 1);
            const uint32_t from = tmem + ((uint32_t)warp << 21) + buf * m.tile_rows;   // lane 32 * warp
            const bool sums = kb0 < kb1;
            if (sums) {
                wait(acc_full(buf), buf_phase, kb1 - kb0);
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
                    if (!dead) narrow_store16<FDT>(a, v, tile.r0 + r, tile.rows - r, f, bias, bias_even, bias_odd);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0 && sums && !dead) mbar_arrive(acc_empty(buf));
            } else {
                // rows of the tile in shares of `share`; share i is finished by CTA i
                const int share = m.tile_rows / m.split;
                meet();
                int owner = 0, at = 0;
                const uint32_t mine = base + (rank * share * 128 + threadIdx.x) * 4;
                uint32_t to = cluster_map(mine, 0);
#pragma unroll 1
                for (int r = 0; r < tile.rows; r += 16) {
                    float v[16];
                    if (sums) {
                        tmem_load16(from + r, v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = 0.0f;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (r + i < tile.rows) st_cluster_f32(to + at * 512, v[i]);
                        if (++at == share) {
                            at = 0;
                            to = cluster_map(mine, min(++owner, m.split - 1));
                        }
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
                    if (!dead) narrow_store16<FDT>(a, v, tile.r0 + r0 + r, min(share - r, tile.rows - r0 - r), f, bias, bias_even, bias_odd);
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
    if (m.split > 1) cluster_sync();   // a CTA's memory stays until the others have stopped using it
    if (warp == 5) {
        tc_fence_after();
        tmem_free<1>(tmem, m.tmem_columns);
    }
}

// ---- launch -------------------------------------------------------------------------------------------------
template <int KIND, int FDT, bool BWD>
static cudaError_t launch_narrow_one(const CUtensorMap &xmap, const CUtensorMap &wmap, const LinearMmaArgs &m, int grid, size_t smem, const LaunchCfg &cfg,
                                     cudaStream_t stream)
{
    static std::atomic<unsigned long long> ready{0};
    return launch_cluster(linear_narrow_kernel<KIND, FDT, BWD>, m.split, NARROW_THREADS, xmap, wmap, m, grid, smem, cfg, stream, ready);
}

template <int FDT, bool BWD>
static cudaError_t launch_narrow_kind(int kind, const CUtensorMap &xmap, const CUtensorMap &wmap, const LinearMmaArgs &m, int grid, size_t smem,
                                      const LaunchCfg &cfg, cudaStream_t stream)
{
    switch (kind) {
    case KIND_PACK8:   // bytes either way
    case KIND_I8: return launch_narrow_one<KIND_I8, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_PACK4: return launch_narrow_one<KIND_PACK4, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_PACK2: return launch_narrow_one<KIND_PACK2, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_E2M1: return launch_narrow_one<KIND_E2M1, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_E4M3: return launch_narrow_one<KIND_E4M3, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    case KIND_E5M2: return launch_narrow_one<KIND_E5M2, FDT, BWD>(xmap, wmap, m, grid, smem, cfg, stream);
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace qk
