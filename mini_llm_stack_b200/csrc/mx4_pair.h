// The product of many rows by pairs of blocks: two neighbouring SMs work on one tile of 256 rows of the batch (or of an expert)
// by up to NT rows of weights.
//
// At four bits a value an instruction is done with its operands in a third of the time in which L2 brings them to a lone block,
// whose 128 x 192 tile asks for 43 KB for every 256 of K.  Here a block brings in its 128 rows of the batch and half of the
// tile's weights (31 KB for 128 x 192, 35 for 128 x 256), and the instruction, issued by the first block of the pair, takes
// both halves.  Each block holds the scales of its own rows and of all the tile's weights.
//
// The batch's rows lie on the 128-row side: a thread of the epilogue then holds neighbouring outputs of one row, gate and up of
// the same output among them, and stores whole sectors of 32 bytes, or with a transposition between four threads lines of 128.
// (With the weights there, a warp's stores are 64 or 128 bytes of a row each: 2,048 rows x 28,672 x 4,096 with SwiGLU took 213 us
// instead of 95, 110 of them the epilogue.)
//
// Tensor memory: ACC_COLS columns of accumulators, every second one from the first column on, the others up to the last, so that
// two that fit beside one another overlap: the epilogue of one lies under the instructions of the next.  NT = 192 always fits;
// one of 256 asks for fewer bytes, but waits until half of the one before it has been read: the half that it takes, which is
// read first.  Behind them the scales of the last SF_SLOTS stages.
//
// Hand-overs inside the pair, as in the bfloat16 product: full[s] (first block) counts both blocks' copies; empty[s] and acc_full[a]
// arrive on both blocks' barriers; acc_free[a] and acc_empty[a] (first block) take the arrivals of both blocks' epilogue warps,
// when they have read the half of an accumulator that the next may take, and all of it.  No load is multicast.
//
// These kernels are launched plainly.  Chained behind a quantisation whose blocks came in several rounds and let their successors start
// at once, a run under a profiler did not end; what it waited for, reading did not show.  (Without a bound are the allocation of
// tensor memory, the wait for the kernels in front and the cluster's barriers, and at those every thread arrives whatever ran out
// before.)  Nothing stands in that place any more: such a quantisation lets nobody start early (mx4.cu, `at_once`).
//
// What bounds it: operands out of L2 (2,048 x 14,336 by 4,096 in 44 us, 5.5 PFLOP/s; 2,048 tokens, six of 64 experts, gate and up
// 2 x 1,408 of 4,096 in 100 us, 70 without copies), and where float32 sums of slots are stored, memory (down 1,408 by 4,096 in 84 us
// for 450 MB).
#pragma once
#include "mx4_gemm.h"

namespace mls_mx4 {

// A box of a 3-D tensor map, from either block of a pair, that completes on the first one's barrier.
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .b32 rbar;\n\t"
        "mapa.shared::cluster.u32 rbar, %2, 0;\n\t"
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [rbar];\n\t}"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

template <int NT_>
struct PairPlan {
    static constexpr int NT = NT_, ROWS = 2 * UMMA_M;
    static constexpr int A_BYTES = UMMA_M * CODE_ROW, B_BYTES = NT / 2 * CODE_ROW;
    static constexpr int SF_A = A_BYTES + B_BYTES, SF_B = SF_A + SF_STAGE;
    static constexpr int STAGE = SF_B + 2 * SF_STAGE;
    static constexpr int STAGES = (220 * 1024) / STAGE;
    static constexpr int SF_SLOT_COLS = 3 * SF_COLS;
    static constexpr int ACC_COLS = 384;
    static constexpr int FIT = (512 - ACC_COLS) / SF_SLOT_COLS;
    static constexpr int SF_SLOTS = FIT < STAGES ? FIT : STAGES;
    static constexpr int SETS = NT / 64;                           // of four epilogue warps
    static constexpr int THREADS = 64 + 128 * SETS;
    static constexpr int BARS = STAGES * STAGE;                    // full, empty [STAGES]; acc_full, acc_free, acc_empty [2]
    static constexpr int TMEM_SLOT = BARS + 8 * (2 * STAGES + 6);
    static constexpr int TABLE = TMEM_SLOT + 16;
    static constexpr int FIXED = TABLE + 1024;
    static_assert(ACC_COLS + SF_SLOTS * SF_SLOT_COLS <= 512 && STAGE % 1024 == 0 && ACC_COLS >= NT &&
                  FIXED + 4 * (TABLE_EXPERTS + 1) <= 227 * 1024, "tile");
};

// 32 bytes of a row at a 32-byte place: whole sectors, where a warp's lanes store to 32 rows.
__device__ __forceinline__ void store32(void* at, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n"
                 ::"l"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
// COUNT neighbouring outputs of a row, `there` of which exist, at a 32-byte place.
template <typename OUT, int COUNT>
__device__ __forceinline__ void store_run(OUT* out, const float (&v)[COUNT], int there) {
    constexpr int PER = 32 / sizeof(OUT);
    if (there >= COUNT) {
#pragma unroll
        for (int i = 0; i < COUNT / PER; ++i) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (sizeof(OUT) == 2) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v[PER * i + 2 * j], v[PER * i + 2 * j + 1]);
                    memcpy(&w[j], &h, 4);
                } else {
                    w[j] = __float_as_uint(v[PER * i + j]);
                }
            }
            store32(out + PER * i, w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < COUNT; ++i)
            if (i < there) Elem<OUT>::store(out + i, v[i]);
    }
}

// 16 neighbouring outputs of the rows of a warp's lanes, at places that suit no wide store: turned within each half of the warp,
// so that a store takes 16 neighbours of two rows.  (A lane's one by one: 143 us for 2,000 x 14,000 by 3,999 instead of 60.)
template <typename OUT>
__device__ __forceinline__ void store_turned(OUT* out, int width, const float (&v)[16], int col, int to, bool mine, int lane) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i]);
#pragma unroll
    for (int bit = 1; bit < 16; bit *= 2) {
        const bool upper = lane & bit;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i & bit) continue;
            const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? w[i] : w[i | bit], bit);
            (upper ? w[i] : w[i | bit]) = got;
        }
    }
    const int n = col + (lane & 15), row = mine ? to : -1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {                   // the lane's column of row i of its half
        const int r = __shfl_sync(0xffffffffu, row, (lane & 16) + i);
        if (r >= 0 && n < width) Elem<OUT>::store(out + (size_t)r * width + n, __uint_as_float(w[i]));
    }
}

// 16 lanes of tensor memory x 32 columns: thread t gets, for i < 4, columns 8 i + 2 (t % 4) and the one behind it of lane t / 4 in
// r[4 i], r[4 i + 1] and of lane t / 4 + 8 in r[4 i + 2], r[4 i + 3].
__device__ __forceinline__ void tmem_ld_16x32(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
// Of four threads that hold columns 8 i + 2 t, 8 i + 2 t + 1 (i < 4; t: which of the four) in v[i], thread t gets columns 8 t to 8 t + 7:
// a 4 x 4 transposition of pairs, by halves.
__device__ __forceinline__ void gather_columns(uint32_t (&v)[4][2], int t) {
#pragma unroll
    for (int bit = 1; bit < 4; bit *= 2) {
        const bool upper = t & bit;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i & bit) continue;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? v[i][x] : v[i | bit][x], bit);
                (upper ? v[i][x] : v[i | bit][x]) = got;
            }
        }
    }
}

// What a warp knows of the rows that it stores.  Whole lines (store_lines): thread t stores to the rows t / 4 + 8 z; else its lane's.
struct To {
    int row[4];
    float share[4];
    bool mine[4];
};
// The same runs for outputs of 32 bits that need no neighbours: a warp stores 128 bytes each to eight rows at a time (32 bytes
// each to its 32 rows: 152 us instead of 146, at the same sizes).
template <typename OUT, bool GROUPED, int RUNS, typename Read>
__device__ __forceinline__ void store_lines(const Product& p, uint32_t d, int set, int sets, bool down, int columns, int n0,
                                            bool any, const To& to, int lane, Read read) {
#pragma unroll 1
    for (int i = 0; i < RUNS; ++i) {
        const int c0 = ((down ? RUNS - 1 - i : i) * sets + set) * 32;
        if (!any || c0 >= columns) {                 // (nothing to read)
            read(i);
            continue;
        }
        uint32_t x[2][16];
        tmem_ld_16x32(d + c0, x[0]);
        tmem_ld_16x32(d + (16u << 16) + c0, x[1]);
        tmem_ld_wait();
        read(i);
        const int col = n0 + c0 + lane % 4 * 8;
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            uint32_t w[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j][0] = x[z / 2][4 * j + z % 2 * 2], w[j][1] = x[z / 2][4 * j + z % 2 * 2 + 1];
            gather_columns(w, lane % 4);
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = __uint_as_float(w[j / 2][j % 2]);
                if (GROUPED) v[j] *= to.share[z];
                if (p.unit == RELU2) v[j] = relu_squared(v[j]);
            }
            if (to.mine[z]) store_run<OUT>((OUT*)p.out + (size_t)to.row[z] * p.width + col, v, p.width - col);
        }
    }
}

// A warp's runs of 32 columns of the accumulator, for its 32 rows: this thread's goes to row `to`.  The set's runs lie `step`
// columns apart, in the order in which they are to be read; `read(i)` is called behind the i-th one's reading.
template <typename OUT, bool GROUPED, int RUNS, bool VEC, typename Read>
__device__ __forceinline__ void store_rows(const Product& p, uint32_t d, int set, int sets, bool down, int columns, int n0,
                                           bool any, bool mine, int to, float share, int lane, Read read) {
    OUT *out = (OUT*)p.out, *row = out + (size_t)to * p.width;
    const bool pairs = p.unit == GATED, square = p.unit == RELU2;
#pragma unroll 1
    for (int i = 0; i < RUNS; ++i) {
        const int c0 = ((down ? RUNS - 1 - i : i) * sets + set) * 32;
        if (!any || c0 >= columns) {                 // (nothing to read)
            read(i);
            continue;
        }
        uint32_t x[16], y[16];
        tmem_ld16(d + c0, x);
        tmem_ld16(d + c0 + 16, y);
        tmem_ld_wait();
        read(i);
        if (pairs) {
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                float g = __uint_as_float(x[j]), up = __uint_as_float(y[j]);
                if (GROUPED) g *= share, up *= share;
                v[j] = unit_of_sums<OUT>(g, up, p.alpha, p.limit);
            }
            const int col = (n0 + c0) / 2;
            if (!VEC) store_turned<OUT>(out, p.width, v, col, to, mine, lane);
            else if (mine) store_run<OUT>(row + col, v, p.width - col);
        } else {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    v[j] = __uint_as_float(half ? y[j] : x[j]);
                    if (GROUPED) v[j] *= share;
                    if (square) v[j] = relu_squared(v[j]);
                }
                const int col = n0 + c0 + 16 * half;
                if (!VEC) store_turned<OUT>(out, p.width, v, col, to, mine, lane);
                else if (mine) store_run<OUT>(row + col, v, p.width - col);
            }
        }
    }
}

template <int NT_, bool GROUPED>
__device__ __forceinline__ void pair_block(const Product& p, const CUtensorMap* rows_map, const CUtensorMap* half_map,
                                           const CUtensorMap* w_map, const CUtensorMap* sf_rows_map, const CUtensorMap* sf_w_map) {
    using L = PairPlan<NT_>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - raw);
    auto full = [&](int s) { return base + L::BARS + 8u * s; };
    auto empty = [&](int s) { return base + L::BARS + 8u * (L::STAGES + s); };
    auto acc_full = [&](int a) { return base + L::BARS + 8u * (2 * L::STAGES + a); };
    auto acc_free = [&](int a) { return base + L::BARS + 8u * (2 * L::STAGES + 2 + a); };
    auto acc_empty = [&](int a) { return base + L::BARS + 8u * (2 * L::STAGES + 4 + a); };
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + L::TMEM_SLOT);
    int* start = reinterpret_cast<int*>(gbase + L::TABLE);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();                          // 0: issues the instructions
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full(a), 1);
            mbar_init(acc_free(a), 2 * 4 * L::SETS);
            mbar_init(acc_empty(a), 2 * 4 * L::SETS);
        }
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        chain_release();                 // (not before: see there)
    }
    chain_wait();
    if (GROUPED && warp == 0) row_tiles<L::ROWS>(p, lane, start);
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();                  // both blocks' barriers, tables and tensor memory are ready
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int w_tiles = (p.N + L::NT - 1) / L::NT, sf_tiles = (p.N + TILE_ROWS - 1) / TILE_ROWS;
    const int units = (GROUPED ? start[p.n_experts] : (p.M + L::ROWS - 1) / L::ROWS) * w_tiles;
    const int kblocks = (p.K + BK - 1) / BK;
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
    bool timed_out = false;
    // the accumulator's columns, up to a multiple of 32 (a half of the weights comes from each block), and where they are
    auto columns = [&](const Unit& u) { return (min(L::NT, p.N - u.n0) + 31) & ~31; };
    auto place = [&](const Unit& u, int it) { return it & 1 ? L::ACC_COLS - columns(u) : 0; };

    if (warp == 0) {
        // ----------------------------------------------------------------- TMA producer
        if (lane == 0) {
            int g = 0;
            for (int i = first; i < units && !timed_out; i += step) {
                const Unit u = unit_of<L::ROWS, GROUPED, L::NT>(p, i, w_tiles, start);
                // (a second block without rows brings in none, one with up to 64 half a tile: what else lies in the stage ends in
                // sums that nobody reads)
                auto row_bytes = [&](int block) {
                    const int rows = u.rows - block * UMMA_M;
                    return rows <= 0 ? 0 : GROUPED && rows <= UMMA_M / 2 ? L::A_BYTES / 2 : L::A_BYTES;
                };
                const int mine = row_bytes((int)rank);
                const CUtensorMap* from = mine == L::A_BYTES ? rows_map : half_map;
                const uint32_t bytes = row_bytes(0) + row_bytes(1) + 2 * (L::B_BYTES + 3 * SF_STAGE);
                const int row = u.row0 + (int)rank * UMMA_M, w_row = u.e * p.N + u.n0 + (int)rank * (columns(u) / 2);
                const int sf_row = u.sf_tile + (int)rank, sf_w = u.e * sf_tiles + u.n0 / TILE_ROWS;
                for (int kb = 0; kb < kblocks; ++kb, ++g) {
                    const int slot = g % L::STAGES;
                    if (!mbar_wait(empty(slot), ((g / L::STAGES) & 1) ^ 1)) {
                        timed_out = true;
                        break;
                    }
                    const uint32_t a = base + slot * L::STAGE, bar = full(slot);
                    // both blocks' copies of the stage complete on the first one's barrier
                    if (rank == 0) mbar_arrive_expect_tx(bar, bytes);
                    if (mine) tma_load_2d_pair(a, from, kb * CODE_ROW, row, bar);
                    tma_load_2d_pair(a + L::A_BYTES, w_map, kb * CODE_ROW, w_row, bar);
                    tma_load_3d_pair(a + L::SF_A, sf_rows_map, 0, kb, sf_row, bar);
                    tma_load_3d_pair(a + L::SF_B, sf_w_map, 0, kb, sf_w, bar);
                }
            }
            // the copies under way land before the pair's shared memory goes away (the first block's barriers count both
            // blocks' bytes, and both blocks meet once more)
            if (rank == 0)
                for (int j = g > L::STAGES ? g - L::STAGES : 0; j < g; ++j)
                    if (!mbar_wait_cluster(full(j % L::STAGES), (j / L::STAGES) & 1)) timed_out = true;
        }
    } else if (warp == 1) {
        if (rank == 0) {
            // ---------------------------------------------------- instructions, for the pair
            // What a stage costs this warp beside the instructions bounds tiles of few columns: 0.39 us a stage with the
            // places of slots divided out anew and waits one by one, 0.28 now; the instructions of 256 columns take 0.33.
            constexpr bool FEWER = L::SF_SLOTS < L::STAGES;
            const uint64_t first_a = umma_desc(base), first_sf = atom_desc(base + L::SF_A);
            int it = 0, columns_before = 0, slot = 0, phase = 0;
            int sf_slot = 0, old = L::STAGES - L::SF_SLOTS, old_phase = 1;      // (the phase before the first is over)
            for (int i = first; i < units && !timed_out; i += step, ++it) {
                const Unit u = unit_of<L::ROWS, GROUPED, L::NT>(p, i, w_tiles, start);
                const int n = columns(u), acc = it & 1;
                const uint32_t idesc0 = idesc_mx4(2 * UMMA_M, n, 0), idesc1 = idesc_mx4(2 * UMMA_M, n, 1);
                // the accumulator before the last has been read, and of the last the columns that this one may take, where
                // it does not fit beside it
                if (!mbar_wait_cluster_warp(acc_empty(acc), ((it >> 1) & 1) ^ 1) ||
                    (columns_before + n > L::ACC_COLS &&
                     !mbar_wait_cluster_warp(acc_free(acc ^ 1), ((it - 1) >> 1) & 1))) {
                    timed_out = true;
                    break;
                }
                columns_before = n;
                const uint32_t d = tmem_base + place(u, it), shift = u.n0 % TILE_ROWS / 32;
                int left = p.K;
                for (int kb = 0; kb < kblocks; ++kb, left -= BK) {
                    // the stage is there, and the instructions that read its scales' columns last are done: both asked at
                    // once, one by one only where one of them is not
                    bool ready = mbar_try_wait_cluster(full(slot), phase);
                    if (FEWER) ready &= mbar_try_wait(empty(old), old_phase);
                    if (!__all_sync(0xffffffffu, ready) &&
                        (!mbar_wait_cluster_warp(full(slot), phase) || (FEWER && !mbar_wait_warp(empty(old), old_phase)))) {
                        timed_out = true;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sf = tmem_base + L::ACC_COLS + sf_slot * L::SF_SLOT_COLS;
                    const uint64_t a = first_a + slot * (L::STAGE >> 4), scales = first_sf + slot * (L::STAGE >> 4);
                    if (elect_one()) {
                        copy_scales<true, 2>(sf, sf + SF_COLS, scales, scales + (SF_STAGE >> 4));
                        multiply_stage<true, 2>(d, a, a + (L::A_BYTES >> 4), idesc0, idesc1, sf, sf + SF_COLS + shift, kb > 0,
                                                left >= BK ? 4 : (left + 63) / 64);
                        umma_commit_pair(empty(slot), 3);          // both blocks' stage is free
                    }
                    __syncwarp();
                    if (++slot == L::STAGES) slot = 0, phase ^= 1;
                    if (++sf_slot == L::SF_SLOTS) sf_slot = 0;
                    if (++old == L::STAGES) old = 0, old_phase ^= 1;
                }
                if (elect_one()) umma_commit_pair(acc_full(acc), 3);   // both blocks' accumulator is complete
                __syncwarp();
            }
        }
    } else {
        // -------------------------------------------------------------------- epilogue
        const int q = warp & 3, set = (warp - 2) >> 2;
        // two runs of 32 columns a set: the first of 256 in the columns that the next accumulator may take
        constexpr int RUNS = L::NT / 32 / L::SETS, FREE_AT = L::NT == 256 ? RUNS / 2 - 1 : RUNS - 1;
        const bool vec = p.width % (p.out_type == MLS_BF16 ? 16 : 8) == 0 && reinterpret_cast<uintptr_t>(p.out) % 32 == 0;
        // Relaxed is enough: what is handed over are columns of tensor memory, nothing in ordinary memory.  PTX orders tensor-memory
        // operations of different threads by wait::ld (of the whole warp, as the load: lane 0's are the warp's),
        // fence::before_thread_sync and an arrival on one side, a wait for it and fence::after_thread_sync on the other, and gives
        // that pattern with relaxed arrivals of the cluster's scope; the wait here even acquires.  A release would wait for the
        // stores of the runs before as well: 22.5 us instead of 18.9 for 707 rows x 2,048 by 16,384 gated sums.
        auto arrive = [&](uint32_t bar) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote_relaxed(bar, 0);
        };
        // Where this thread's rows go and the weights of their slots: numbers of slots read two units ahead, weights one, while
        // instructions run and sums are stored (read when their unit's turn came: 146 us instead of 129 for 2,048 tokens down, six
        // chosen of 64 experts of 4,096 x 1,408)
        const bool lines = p.unit != GATED && p.out_type != MLS_BF16 && vec, look = GROUPED && (p.unit == DOWN || p.scale);
        const int row = (int)rank * UMMA_M + q * 32;               // the warp's first
        auto row_of = [&](int z) { return row + (lines ? lane / 4 + 8 * z : lane); };
        auto unit_at = [&](int i) {
            Unit u = {};                                           // (behind the last: no rows)
            if (i < units) u = unit_of<L::ROWS, GROUPED, L::NT>(p, i, w_tiles, start);
            return u;
        };
        struct Slots {
            int at[4];
        };
        auto slots_of = [&](const Unit& u) {
            Slots s;
#pragma unroll
            for (int z = 0; z < 4; ++z)
                s.at[z] = look && (z == 0 || lines) && row_of(z) < u.rows ? p.order[u.row0 + row_of(z)] : 0;
            return s;
        };
        struct Shares {
            float at[4];
        };
        auto shares_of = [&](const Unit& u, const Slots& s) {
            Shares f;
#pragma unroll
            for (int z = 0; z < 4; ++z)
                f.at[z] = look && p.scale && (z == 0 || lines) && row_of(z) < u.rows ? p.weight[s.at[z]] : 1.f;
            return f;
        };
        Unit u = unit_at(first), u1 = unit_at(first + step);
        Slots slots = slots_of(u), slots1 = slots_of(u1);
        Shares shares = shares_of(u, slots);
        int it = 0;
        for (int i = first; i < units; i += step, ++it) {
            const Unit u2 = unit_at(i + 2 * step);
            const Slots slots2 = slots_of(u2);
            const Shares shares1 = shares_of(u1, slots1);
            const int acc = it & 1;
            // (the columns in the middle first: an accumulator at the end begins there, one at the start ends there)
            const bool down = acc == 0;
            const uint32_t d = tmem_base + place(u, it);
            auto read = [&](int run) {
                if (run == FREE_AT) arrive(acc_free(acc));
                if (run == RUNS - 1) arrive(acc_empty(acc));
            };
            const bool any = row < u.rows;
            To to;
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                to.row[z] = GROUPED && p.unit == DOWN ? slots.at[z] : u.row0 + row_of(z);
                to.share[z] = shares.at[z];
                to.mine[z] = row_of(z) < u.rows;
            }
            if (!mbar_wait_warp(acc_full(acc), (it >> 1) & 1)) {
                timed_out = true;
                break;
            }
            tc_fence_after();
            const uint32_t at = d + ((uint32_t)(q * 32) << 16);
            if (lines)
                store_lines<float, GROUPED, RUNS>(p, at, set, L::SETS, down, columns(u), u.n0, any, to, lane, read);
            else if (vec && p.out_type == MLS_BF16)
                store_rows<__nv_bfloat16, GROUPED, RUNS, true>(p, at, set, L::SETS, down, columns(u), u.n0, any, to.mine[0],
                                                               to.row[0], to.share[0], lane, read);
            else if (p.out_type == MLS_BF16)
                store_rows<__nv_bfloat16, GROUPED, RUNS, false>(p, at, set, L::SETS, down, columns(u), u.n0, any, to.mine[0],
                                                                to.row[0], to.share[0], lane, read);
            else if (vec)
                store_rows<float, GROUPED, RUNS, true>(p, at, set, L::SETS, down, columns(u), u.n0, any, to.mine[0], to.row[0],
                                                       to.share[0], lane, read);
            else
                store_rows<float, GROUPED, RUNS, false>(p, at, set, L::SETS, down, columns(u), u.n0, any, to.mine[0], to.row[0],
                                                        to.share[0], lane, read);
            u = u1, u1 = u2, slots = slots1, slots1 = slots2, shares = shares1;
        }
    }
    if (timed_out && p.status) atomicOr(p.status, MLS_STATUS_TIMEOUT);
    __syncwarp();
    tc_fence_before();
    cluster_sync_all();                  // nobody of the pair touches tensor memory any more
    if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}
}  // namespace mls_mx4
