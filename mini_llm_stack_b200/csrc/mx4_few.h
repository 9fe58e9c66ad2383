// A product of few rows by 4-bit microscaled weights, in one kernel from the rows to the outputs.
//
// Such a product is a stream of weights.  A block takes 128 of their rows (an instruction's) and a slice of K; the blocks
// of a tile's slices form a cluster of up to eight.  With FUSED, while the first weights are on their way, eight warps quantise the
// slice of the rows straight into the layout that the instructions read; without, the rows' codes and scales come with
// the weights' from memory.  The slices' sums meet in shared memory: every block adds up its share of the tile over the
// cluster, in the order of the slices, and stores it.
#pragma once
#include "mx4_gemm.h"

namespace mls_mx4 {

constexpr int FEW_STAGES = 4;
constexpr int FEW_WORKERS = 8;                        // warps that quantise, read the sums and store them
constexpr int FEW_THREADS = 32 * (2 + FEW_WORKERS);
constexpr int FEW_SLICES = 8;                         // blocks of a cluster, at most
// The least shared memory of a block: four of them fill an SM, so that the 128 columns of tensor memory that each holds are always
// there.  Blocks of a cluster hold them while they wait for one another; with more blocks than columns two clusters
// could each wait for what the other has.  Nor do they fit beside a pair of blocks of this or the bfloat16 product, which wait for
// each other in the same way and hold every column.
constexpr int FEW_LEAST = 48 * 1024;
constexpr int FEW_SLICE = 12;                         // stages of K of a slice, at most (FUSED: two blocks an SM)

struct FewProduct {
    const void* rows;                                 // [M, K], row stride ld (FUSED)
    void* out;                                        // [M, width]
    const uint8_t *sf_w, *sf_a;
    long long ld;
    int rows_type, vec, unit, out_type;
    int M, N, K, width;
    int slice;                                        // stages of 256 of K a block takes
    int early;                                        // no kernel under way writes the weights
    float alpha, limit;
    int* status;
};

// NR: rows of the batch an instruction takes.
template <int NR, bool FUSED>
struct FewPlan {
    static constexpr int ROWS_STAGE = NR * CODE_ROW + SF_STAGE;
    static constexpr int A_STAGE = UMMA_M * CODE_ROW + SF_STAGE;
    static constexpr int STAGE = A_STAGE + (FUSED ? 0 : ROWS_STAGE);
    static constexpr int SF_COLS_STAGE = 2 * SF_COLS;
    static constexpr int SF_AT = NR;
    static constexpr int COLS = pow2_at_least(SF_AT + FEW_STAGES * SF_COLS_STAGE);
    static_assert(COLS * (227 * 1024 / FEW_LEAST) <= 512, "tensor memory of the blocks that fit an SM");
    // a slice's stages (as many as it has, up to FEW_STAGES), FUSED its rows' codes and scales, barriers.  The sums
    // [NR][128] take the place of the stages, once the instructions are done.
    __host__ __device__ static constexpr int stages(int slice) { return slice < FEW_STAGES ? slice : FEW_STAGES; }
    __host__ __device__ static constexpr int rows(int slice) { return stages(slice) * STAGE; }
    __host__ __device__ static constexpr int bars(int slice) {
        const int loads = rows(slice) + (FUSED ? slice * ROWS_STAGE : 0), sums = NR * UMMA_M * 4;
        return loads > sums ? loads : sums;
    }
    __host__ __device__ static constexpr int total(int slice) {
        const int bytes = bars(slice) + 8 * (2 * FEW_STAGES + 2) + 16 + 1024;
        return bytes > FEW_LEAST ? bytes : FEW_LEAST;
    }
};

__device__ __forceinline__ float load_cluster_f32(uint32_t addr, uint32_t cta) {
    float v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f32 %0, [r];\n\t}"
                 : "=f"(v) : "r"(addr), "r"(cta));
    return v;
}

template <typename T, bool VEC, int NR>
__device__ __forceinline__ void quantise_slice(const FewProduct& p, int kb0, int n_kb, int worker, int lane, uint8_t* rows) {
    using L = FewPlan<NR, true>;
    // a warp's task: 256 values of a row; warps take them in turn, rows fastest
    const T *x = (const T*)p.rows, *end = x + (p.M - 1) * p.ld + p.K;
    const int step_kb = FEW_WORKERS / p.M, step_r = FEW_WORKERS - step_kb * p.M;
    int kb = worker / p.M, r = worker - kb * p.M;
    constexpr int AT_ONCE = 4;
    while (kb < n_kb) {
        Raw<T, VEC, 1> raw[AT_ONCE];
        int at_kb[AT_ONCE], at_r[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            at_kb[j] = kb, at_r[j] = r;
            if (kb < n_kb) load_raw(x, end, x + r * p.ld, (kb0 + kb) * BK + lane * 8, p.K, raw[j]);
            kb += step_kb, r += step_r;
            if (r >= p.M) r -= p.M, ++kb;
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            if (at_kb[j] >= n_kb) break;
            Eight<T> held[1];
            settle(raw[j], x + at_r[j] * p.ld, (kb0 + at_kb[j]) * BK + lane * 8, p.K, held);
            uint32_t scales, codes[1];
            quantize_lane(held, lane, codes, scales);
            uint8_t* stage = rows + at_kb[j] * L::ROWS_STAGE;
            // (the 128-byte swizzle: a row's 16-byte pieces change places by the row's number)
            *reinterpret_cast<uint32_t*>(stage + at_r[j] * CODE_ROW + (((lane >> 2) ^ (at_r[j] & 7)) << 4) + (lane & 3) * 4) =
                codes[0];
            if ((lane & 15) == 0)
                *reinterpret_cast<uint32_t*>(stage + NR * CODE_ROW + (lane >> 4) * ATOM + row_in_atom(at_r[j])) = scales;
        }
    }
}

// Block (slice, tile) of the grid; the slices of a tile are a cluster.
template <int NR, bool FUSED>
__device__ __forceinline__ void few_block(const FewProduct& p, const CUtensorMap* rows_map, const CUtensorMap* w_map) {
    using L = FewPlan<NR, FUSED>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - raw);
    const int bars = L::bars(p.slice), stages = L::stages(p.slice);
    auto full = [&](int s) { return base + bars + 8u * s; };
    auto empty = [&](int s) { return base + bars + 8u * (FEW_STAGES + s); };
    const uint32_t rows_full = base + bars + 8u * (2 * FEW_STAGES), acc_full = rows_full + 8u;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + bars + 8 * (2 * FEW_STAGES + 2));

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < FEW_STAGES; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        mbar_init(rows_full, FEW_WORKERS);
        mbar_init(acc_full, 1);
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), L::COLS);
        chain_release();                 // (not before: see there)
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int kblocks = (p.K + BK - 1) / BK;
    const int kb0 = blockIdx.x * p.slice, n_kb = max(0, min(p.slice, kblocks - kb0));
    const int n0 = blockIdx.y * UMMA_M;
    bool timed_out = false;

    if (warp == 0) {
        // ----------------------------------------------------------------- TMA producer
        if (lane == 0) {
            const uint8_t* sf_w = p.sf_w + ((size_t)blockIdx.y * kblocks + kb0) * SF_STAGE;
            const uint8_t* sf_a = FUSED ? nullptr : p.sf_a + (size_t)kb0 * SF_STAGE;
            auto load_weights = [&](int j) {
                const uint32_t a = base + j % stages * L::STAGE, bar = full(j % stages);
                mbar_arrive_expect_tx(bar, L::STAGE);
                tma_load_2d(a, w_map, (kb0 + j) * CODE_ROW, n0, bar);
                bulk_load_1d(a + UMMA_M * CODE_ROW, sf_w + (size_t)j * SF_STAGE, SF_STAGE, bar);
            };
            auto load_rows = [&](int j) {
                const uint32_t b = base + j % stages * L::STAGE + L::A_STAGE, bar = full(j % stages);
                tma_load_2d(b, rows_map, (kb0 + j) * CODE_ROW, 0, bar);
                bulk_load_1d(b + NR * CODE_ROW, sf_a + (size_t)j * SF_STAGE, SF_STAGE, bar);
            };
            // (weights that nobody writes are asked for while the kernel before this one may still run)
            const int ahead = min(n_kb, stages);
            if (!p.early) chain_wait();
            for (int j = 0; j < ahead; ++j) load_weights(j);
            if (p.early) chain_wait();
            if (!FUSED)
                for (int j = 0; j < ahead; ++j) load_rows(j);
            int g = ahead;
            for (; g < n_kb; ++g) {
                if (!mbar_wait(empty(g % stages), ((g / stages) & 1) ^ 1)) {
                    timed_out = true;
                    break;
                }
                load_weights(g);
                if (!FUSED) load_rows(g);
            }
            // the copies under way land before the block's shared memory goes away
            for (int j = g > stages ? g - stages : 0; j < g; ++j)
                if (!mbar_wait(full(j % stages), (j / stages) & 1)) timed_out = true;
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- instructions
        const uint32_t idesc0 = idesc_mx4(UMMA_M, NR, 0), idesc1 = idesc_mx4(UMMA_M, NR, 1);
        chain_wait();                    // (the kernel before may take longer than a wait for the rows has)
        if (FUSED && !mbar_wait_warp(rows_full, 0)) timed_out = true;
        for (int g = 0; g < n_kb && !timed_out; ++g) {
            const int slot = g % stages;
            if (!mbar_wait_warp(full(slot), (g / stages) & 1)) {
                timed_out = true;
                break;
            }
            tc_fence_after();
            const uint32_t a = base + slot * L::STAGE;
            const uint32_t b = FUSED ? base + L::rows(p.slice) + g * L::ROWS_STAGE : a + L::A_STAGE;
            const uint32_t sf_a = tmem_base + L::SF_AT + slot * L::SF_COLS_STAGE, sf_b = sf_a + SF_COLS;
            const int steps = min(4, (p.K - (kb0 + g) * BK + 63) / 64);
            if (elect_one()) {
                copy_scales<false, 1>(sf_a, sf_b, atom_desc(a + UMMA_M * CODE_ROW), atom_desc(b + NR * CODE_ROW));
                multiply_stage<false, 1>(tmem_base, umma_desc(a), umma_desc(b), idesc0, idesc1, sf_a, sf_b, g > 0, steps);
                umma_commit(empty(slot));
            }
            __syncwarp();
        }
        if (elect_one()) umma_commit(acc_full);
        __syncwarp();
    } else {
        // --------------------------------------------------- the rows, then the sums of the slice
        chain_wait();
        const int worker = warp - 2;
        if (FUSED) {
            uint8_t* rows = gbase + L::rows(p.slice);
            if (p.rows_type == MLS_BF16) {
                if (p.vec) quantise_slice<__nv_bfloat16, true, NR>(p, kb0, n_kb, worker, lane, rows);
                else quantise_slice<__nv_bfloat16, false, NR>(p, kb0, n_kb, worker, lane, rows);
            } else {
                if (p.vec) quantise_slice<float, true, NR>(p, kb0, n_kb, worker, lane, rows);
                else quantise_slice<float, false, NR>(p, kb0, n_kb, worker, lane, rows);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(rows_full);
        }
        if (!mbar_wait_warp(acc_full, 0)) timed_out = true;
        tc_fence_after();
        const int q = warp & 3, half = worker >> 2;
        float* sums = reinterpret_cast<float*>(gbase);
        for (int c0 = half * 16; c0 < NR; c0 += 32) {
            uint32_t v[16];
            tmem_ld16(tmem_base + ((uint32_t)(q * 32) << 16) + c0, v);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 16; ++x)
                // (a slice behind K's end has no instructions, its accumulator no sums)
                sums[(c0 + x) * UMMA_M + q * 32 + lane] = n_kb > 0 ? __uint_as_float(v[x]) : 0.f;
        }
    }
    if (timed_out && p.status) atomicOr(p.status, MLS_STATUS_TIMEOUT);
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();
    if (warp == 1) tmem_dealloc(tmem_base, L::COLS);
    if (warp >= 2) {
        const bool pairs = p.unit == GATED;
        const int per_row = pairs ? UMMA_M / 2 : UMMA_M, count = p.M * per_row, slices = gridDim.x;
        const uint32_t sums = base;
        for (int i = blockIdx.x * (32 * FEW_WORKERS) + threadIdx.x - 64; i < count; i += slices * (32 * FEW_WORKERS)) {
            const int r = i / per_row, j = i - r * per_row;
            const int n = (pairs ? n0 / 2 : n0) + j;
            if (n >= p.width) continue;
            const uint32_t at = sums + 4 * (r * UMMA_M + (pairs ? (j / 16) * 32 + j % 16 : j));
            // (all slices' sums are on their way before the first is added)
            float v = 0.f, u = 0.f, vs[FEW_SLICES], us[FEW_SLICES];
#pragma unroll
            for (int s = 0; s < FEW_SLICES; ++s) {
                if (s < slices) vs[s] = load_cluster_f32(at, s);
                if (s < slices && pairs) us[s] = load_cluster_f32(at + 64, s);
            }
#pragma unroll
            for (int s = 0; s < FEW_SLICES; ++s) {
                if (s < slices) v += vs[s];
                if (s < slices && pairs) u += us[s];
            }
            if (pairs) v = p.out_type == MLS_BF16 ? unit_of_sums<__nv_bfloat16>(v, u, p.alpha, p.limit)
                                                  : unit_of_sums<float>(v, u, p.alpha, p.limit);
            else if (p.unit == RELU2) v = relu_squared(v);
            store_from_float(p.out, (size_t)r * p.width + n, p.out_type, v);
        }
    }
    __syncwarp();
    cluster_sync_all();                  // nobody leaves while its sums are being read
}
}  // namespace mls_mx4
