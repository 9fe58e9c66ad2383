// Block-scaled tcgen05 instructions for 4-bit operands, and the plan of a tile of the products in mx4_gemm.cu.
//
// An instruction takes 64 of K: 128 rows of A and up to 256 of B, 32 bytes a row, from shared memory in the same
// layout as 16 values of 16 bits (128-byte rows, here 256 of K, with the 128-byte swizzle), and two scales a row
// from tensor memory.  Scales lie there as tcgen05.cp leaves an atom of 512 bytes: row r's four bytes (128 of K) in lane
// r % 32 of column r / 32, repeated in the four quarters of the lanes; the instruction descriptor says which two of the
// four bytes it takes.
#pragma once
#include "experts.h"
#include "mx4.h"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace mls_mx4 {
using namespace mls_tc;
using namespace mls_tma;
using mls_experts::DOWN;
using mls_experts::GATED;
using mls_experts::RELU2;

constexpr int BK = 256;                              // K of a stage: 128 bytes of codes a row, two atoms of scales
constexpr int CODE_ROW = 128;
constexpr int SF_STAGE = 2 * ATOM;                   // a tile's scales in a stage
constexpr int SF_COLS = 8;                           // tensor-memory columns of the same

// e2m1 x e2m1 -> f32 with e8m0 scales, both K-major; half: which two of the four bytes of scales (both operands' alike).
__host__ __device__ constexpr uint32_t idesc_mx4(int m, int n, int half) {
    return ((uint32_t)(2 * half) << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) |
           ((uint32_t)(m >> 4) << 24) | ((uint32_t)(2 * half) << 29);
}
// An atom of scales: 32 rows of 16 bytes, no swizzle.
__device__ __forceinline__ uint64_t atom_desc(uint32_t addr) {
    uint64_t d = 0;
    d |= (uint64_t)((addr & 0x3FFFF) >> 4);
    d |= (uint64_t)1 << 16;                          // leading byte offset (unused: 16 bytes wide)
    d |= (uint64_t)(128 >> 4) << 32;                 // stride byte offset: 8-row groups
    d |= (uint64_t)1 << 46;
    return d;
}
__device__ __forceinline__ void copy_atom(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_mx4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t sf_a, uint32_t sf_b, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sf_a), "r"(sf_b), "r"(accumulate) : "memory");
}

// For a pair of blocks (cta_group::2): both blocks' copies from their own shared memory, one instruction for both.
__device__ __forceinline__ void copy_atom_pair(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_mx4_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                              uint32_t sf_a, uint32_t sf_b, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sf_a), "r"(sf_b), "r"(accumulate) : "memory");
}

// The scales of a stage into tensor memory: A's tile of 128 rows to sf_a, B's TILES to sf_b, sub-columns of 128 of K side by side for
// B.  `scales`: descriptor of A's first atom; B's follow A's.
template <bool PAIR, int TILES>
__device__ __forceinline__ void copy_scales(uint32_t sf_a, uint32_t sf_b, uint64_t scales_a, uint64_t scales_b) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        if (PAIR) copy_atom_pair(sf_a + x * 4, scales_a + x * (ATOM >> 4));
        else copy_atom(sf_a + x * 4, scales_a + x * (ATOM >> 4));
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
            const uint64_t from = scales_b + (j * SF_STAGE + x * ATOM >> 4);
            if (PAIR) copy_atom_pair(sf_b + (x * TILES + j) * 4, from);
            else copy_atom(sf_b + (x * TILES + j) * 4, from);
        }
    }
}
// The instructions of a stage: 64 of K each, `steps` of them (fewer than four only at the end of K), onto d or, at the start, in its
// place.  a, b: descriptors of the operands' first 64 of K.
template <bool PAIR, int TILES>
__device__ __forceinline__ void multiply_stage(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc0, uint32_t idesc1,
                                               uint32_t sf_a, uint32_t sf_b, bool onto, int steps) {
    auto one = [&](int kk) {
        const uint32_t idesc = kk & 1 ? idesc1 : idesc0, sa = sf_a + (kk >> 1) * 4, sb = sf_b + (kk >> 1) * (TILES * 4);
        if (PAIR) umma_mx4_pair(d, a + kk * 2, b + kk * 2, idesc, sa, sb, (onto || kk) ? 1u : 0u);
        else umma_mx4(d, a + kk * 2, b + kk * 2, idesc, sa, sb, (onto || kk) ? 1u : 0u);
    };
    if (steps == 4) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) one(kk);
    } else {
#pragma unroll
        for (int kk = 0; kk < 3; ++kk)
            if (kk < steps) one(kk);
    }
}

constexpr int pow2_at_least(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : 512; }

constexpr int TABLE_EXPERTS = 1024;                  // experts of a launch: their table lies beside the stages
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 32 * (2 + EPI_WARPS);

// NT rows of the batch.  Their first one's place among the 128 of a tile of scales is a multiple of 64: an instruction
// takes the columns of scales from an even one on.
template <int NT_>
struct Plan {
    static constexpr int NT = NT_;
    // tiles of 128 rows that NT rows from a multiple of NT on may touch
    static constexpr int STEP = NT % 128 == 0 ? 128 : 64;
    static constexpr int B_TILES = (128 - STEP + NT + 127) / 128;
    static constexpr int BOX = 64;                                 // rows of a copy
    static constexpr int A_BYTES = UMMA_M * CODE_ROW;
    static constexpr int B_BYTES = NT * CODE_ROW;
    static constexpr int SF_A = A_BYTES + B_BYTES;
    static constexpr int SF_B = SF_A + SF_STAGE;
    static constexpr int STAGE = SF_B + B_TILES * SF_STAGE;
    static constexpr int SF_STAGE_COLS = (1 + B_TILES) * SF_COLS;
    static constexpr int ACCS = 2;                                 // accumulators
    static constexpr int FIT = (216 * 1024) / STAGE;
    static constexpr int FIT_T = (512 - ACCS * NT) / SF_STAGE_COLS;
    static constexpr int STAGES = FIT < FIT_T ? (FIT > 8 ? 8 : FIT) : (FIT_T > 8 ? 8 : FIT_T);
    static constexpr int SF_AT = ACCS * NT;                        // first column of the scales
    static constexpr int COLS = pow2_at_least(SF_AT + STAGES * SF_STAGE_COLS);
    static constexpr int BARS = STAGES * STAGE;
    static constexpr int TMEM_SLOT = BARS + 8 * (2 * STAGES + 2 * ACCS);
    static constexpr int TABLE = TMEM_SLOT + 16;                   // [E + 1] ints follow
    static constexpr int FIXED = TABLE + 1024;                     // + alignment slack
    static_assert(NT % 64 == 0 && STAGES >= 2 && SF_AT + STAGES * SF_STAGE_COLS <= 512 &&
                  FIXED + 4 * (TABLE_EXPERTS + 1) <= 227 * 1024, "tile");
};

struct Product {
    void* out;
    const uint8_t *sf_w, *sf_a;                      // scales of the weights and of the rows
    const int *order, *offsets;                      // a routed step's (nullptr: one matrix)
    const float* weight;
    int unit, scale, out_type;                       // unit: DOWN, GATED, RELU2
    int n_experts, first_expert, all_experts;        // of this launch, of the step
    int M, N, K;                                     // N: rows of a weight matrix, a pair's 32 for 16 outputs
    int width;                                       // outputs of a row
    float alpha, limit;
    int* status;
};

// Unit of work i: expert e, outputs from n0, rows [row0, row0 + rows); the scales of its first row lie in tile sf_tile at
// row sf_row.
struct Unit {
    int e, n0, row0, rows, sf_tile, sf_row;
};
// ROWS: rows of weights of a unit, of which there are m_tiles times as many.
template <int NT, bool GROUPED, int ROWS = UMMA_M>
__device__ __forceinline__ Unit unit_of(const Product& p, int i, int m_tiles, const int* start) {
    if (!GROUPED) {
        const int tiles = (p.M + NT - 1) / NT, m = i / tiles, at = (i - m * tiles) * NT;
        return {0, m * ROWS, at, min(NT, p.M - at), at / TILE_ROWS, at % TILE_ROWS};
    }
    const int q = i / m_tiles;
    int lo = 0, hi = p.n_experts;                    // start[lo] <= q < start[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= q) lo = mid;
        else hi = mid;
    }
    const int tiles = start[lo + 1] - start[lo], j = i - start[lo] * m_tiles;
    const int m = j / tiles, at = (j - m * tiles) * NT;
    const int p0 = p.offsets[lo], count = p.offsets[lo + 1] - p0;
    return {lo, m * ROWS, p0 + at, min(NT, count - at), first_tile(p0, p.first_expert + lo) + at / TILE_ROWS,
            at % TILE_ROWS};
}

// start[e]: row tiles of the experts before e.  A lane takes neighbouring experts, whose loads are under way together.
template <int NT>
__device__ __forceinline__ void row_tiles(const Product& p, int lane, int* start) {
    const int per = (p.n_experts + 31) / 32, e0 = min(lane * per, p.n_experts), e1 = min(e0 + per, p.n_experts);
    int sum = 0, at = e0 < e1 ? p.offsets[e0] : 0;
#pragma unroll 8
    for (int e = e0; e < e1; ++e) {
        const int next = p.offsets[e + 1];
        sum += (next - at + NT - 1) / NT;
        at = next;
    }
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += x;
    }
    if (lane == 31) start[p.n_experts] = before;
    before -= sum;
    at = e0 < e1 ? p.offsets[e0] : 0;
#pragma unroll 8
    for (int e = e0; e < e1; ++e) {
        const int next = p.offsets[e + 1];
        start[e] = before;
        before += (next - at + NT - 1) / NT;
        at = next;
    }
}

// The gated unit on two sums on its way to 16 bits: exponential and reciprocal by the approximations of the special function
// unit.  Relative to the output they are off by about 2^-21 around zero; the exponent's rounding makes that grow with |z|, to
// about 2^-18 where the exponential ends (|z| = 88), a thousandth of the rounding to 2^-8.  (In float32's precision, and by half as
// many warps, the unit kept a product of 2,048 x 2,048 with 16,384 gated sums waiting: 55 us instead of 40.)  Outputs of 32 bits take
// the precise one.
template <typename OUT>
__device__ __forceinline__ float unit_of_sums(float g, float u, float alpha, float limit) {
    if (sizeof(OUT) == 4) return mls_experts::gated_unit(g, u, alpha, limit);
    float z = g;
    if (limit > 0.f) {
        g = at_most(g, limit);
        u = at_most(at_least(u, -limit), limit) + 1.0f;
        z = alpha * g;
    }
    float e, r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return g * r * u;
}

// Where the rows of a warp's runs of 16 go (lane x of the first 16 holds row x), and the weights of their slots: read while the
// instructions still run.
template <int RUNS>
struct Rows {
    int to[RUNS];
    float share[RUNS];
};
template <bool GROUPED, int RUNS>
__device__ __forceinline__ Rows<RUNS> rows_of(const Product& p, const Unit& u, int set, int sets, int lane) {
    Rows<RUNS> r;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
        const int x = (i * sets + set) * 16 + lane;
        r.to[i] = u.row0 + x;
        r.share[i] = 1.f;
        if (GROUPED && (p.unit == DOWN || p.scale) && lane < 16 && x < u.rows) {
            const int s = p.order[r.to[i]];
            if (p.scale) r.share[i] = p.weight[s];
            if (p.unit == DOWN) r.to[i] = s;
        }
    }
    return r;
}
// A unit's sums on their way out: a warp takes the quarter q of the lanes (32 of the 128 rows of weights) and its set's runs of 16
// of the batch's rows.
template <typename OUT, bool GROUPED, int RUNS>
__device__ __forceinline__ void store_unit(const Product& p, const Unit& u, const Rows<RUNS>& rows, uint32_t tmem, int q, int set,
                                           int sets, int lane) {
    const bool pairs = p.unit == GATED;
    // this thread's output
    const int n = pairs ? u.n0 / 2 + q * 16 + (lane & 15) : u.n0 + q * 32 + lane;
    const bool mine = n < p.width;
    OUT* out = (OUT*)p.out + n;
    const uint32_t d = tmem + ((uint32_t)(q * 32) << 16);
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
        const int c0 = (i * sets + set) * 16, there = u.rows - c0;
        if (there <= 0) break;
        uint32_t v[16];
        tmem_ld16(d + c0, v);
        tmem_ld_wait();
        if (GROUPED && p.scale) {
#pragma unroll
            for (int x = 0; x < 16; ++x)
                v[x] = __float_as_uint(__uint_as_float(v[x]) * __shfl_sync(0xffffffffu, rows.share[i], x));
        }
        if (pairs) {
            // lanes 0..15 hold the gate's sums of 16 rows, lanes 16..31 up's of the same outputs: the former take the
            // first eight rows, the latter the others
            const bool upper = lane >= 16;
            OUT* at = out + (size_t)(u.row0 + c0 + (upper ? 8 : 0)) * p.width;
            float val[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const uint32_t others = upper ? v[x] : v[x + 8];
                const float got = __shfl_xor_sync(0xffffffffu, __uint_as_float(others), 16);
                const float own = __uint_as_float(upper ? v[x + 8] : v[x]);
                val[x] = unit_of_sums<OUT>(upper ? got : own, upper ? own : got, p.alpha, p.limit);
            }
#pragma unroll
            for (int x = 0; x < 8; ++x, at += p.width)
                if (mine && (upper ? x + 8 : x) < there) Elem<OUT>::store(at, val[x]);
        } else if (GROUPED && p.unit == DOWN) {
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const int s = __shfl_sync(0xffffffffu, rows.to[i], x);
                if (mine && x < there) Elem<OUT>::store(out + (size_t)s * p.width, __uint_as_float(v[x]));
            }
        } else {
            const bool square = p.unit == RELU2;
            OUT* at = out + (size_t)(u.row0 + c0) * p.width;
#pragma unroll
            for (int x = 0; x < 16; ++x, at += p.width) {
                float val = __uint_as_float(v[x]);
                if (square) val = relu_squared(val);
                if (mine && x < there) Elem<OUT>::store(at, val);
            }
        }
    }
}

// The whole of a block's work: see mx4_gemm.cu.
template <int NT, bool GROUPED>
__device__ __forceinline__ void product_block(const Product& p, const CUtensorMap* rows_map, const CUtensorMap* w_map) {
    using L = Plan<NT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - raw);
    auto full = [&](int s) { return base + L::BARS + 8u * s; };
    auto empty = [&](int s) { return base + L::BARS + 8u * (L::STAGES + s); };
    auto acc_full = [&](int a) { return base + L::BARS + 8u * (2 * L::STAGES + a); };
    auto acc_empty = [&](int a) { return base + L::BARS + 8u * (2 * L::STAGES + L::ACCS + a); };
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + L::TMEM_SLOT);
    int* start = reinterpret_cast<int*>(gbase + L::TABLE);

    // (the warp's number from a shuffle: what follows from it alone may stay in uniform registers, from which the
    // instructions take their operands)
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int a = 0; a < L::ACCS; ++a) {
            mbar_init(acc_full(a), 1);
            mbar_init(acc_empty(a), EPI_WARPS);
        }
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), L::COLS);
        chain_release();                 // (not before: see there)
    }
    chain_wait();
    if (GROUPED && warp == 0) row_tiles<NT>(p, lane, start);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int m_tiles = (p.N + UMMA_M - 1) / UMMA_M;
    const int units = (GROUPED ? start[p.n_experts] : (p.M + NT - 1) / NT) * m_tiles;
    const int kblocks = (p.K + BK - 1) / BK;
    const size_t sf_tile_bytes = (size_t)kblocks * SF_STAGE;
    bool timed_out = false;

    if (warp == 0) {
        // ----------------------------------------------------------------- TMA producer
        if (lane == 0) {
            int g = 0;
            for (int i = blockIdx.x; i < units && !timed_out; i += gridDim.x) {
                const Unit u = unit_of<NT, GROUPED>(p, i, m_tiles, start);
                const int boxes = (u.rows + L::BOX - 1) / L::BOX;
                const int sf_tiles = (u.sf_row + u.rows + TILE_ROWS - 1) / TILE_ROWS;
                const uint32_t bytes = L::A_BYTES + boxes * (L::BOX * CODE_ROW) + (1 + sf_tiles) * SF_STAGE;
                const int w_row = u.e * p.N + u.n0;
                const uint8_t* sf_w = p.sf_w + (size_t)(u.e * m_tiles + u.n0 / UMMA_M) * sf_tile_bytes;
                const uint8_t* sf_a = p.sf_a + (size_t)u.sf_tile * sf_tile_bytes;
                for (int kb = 0; kb < kblocks; ++kb, ++g) {
                    const int slot = g % L::STAGES;
                    if (!mbar_wait(empty(slot), ((g / L::STAGES) & 1) ^ 1)) {
                        timed_out = true;
                        break;
                    }
                    const uint32_t a = base + slot * L::STAGE, b = a + L::A_BYTES;
                    mbar_arrive_expect_tx(full(slot), bytes);
                    tma_load_2d(a, w_map, kb * CODE_ROW, w_row, full(slot));
                    bulk_load_1d(a + L::SF_A, sf_w + (size_t)kb * SF_STAGE, SF_STAGE, full(slot));
                    for (int x = 0; x < boxes; ++x)
                        tma_load_2d(b + x * (L::BOX * CODE_ROW), rows_map, kb * CODE_ROW, u.row0 + x * L::BOX,
                                    full(slot));
                    for (int x = 0; x < sf_tiles; ++x)
                        bulk_load_1d(a + L::SF_B + x * SF_STAGE, sf_a + x * sf_tile_bytes + (size_t)kb * SF_STAGE,
                                     SF_STAGE, full(slot));
                }
            }
            // the copies under way land before the block's shared memory goes away
            for (int j = g > L::STAGES ? g - L::STAGES : 0; j < g; ++j)
                if (!mbar_wait(full(j % L::STAGES), (j / L::STAGES) & 1)) timed_out = true;
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- instructions
        const uint64_t first = umma_desc(base), first_sf = atom_desc(base + L::SF_A);
        int it = 0, slot = 0, phase = 0;
        for (int i = blockIdx.x; i < units && !timed_out; i += gridDim.x, ++it) {
            const Unit u = unit_of<NT, GROUPED>(p, i, m_tiles, start);
            const int n = (u.rows + 15) & ~15;
            const uint32_t idesc0 = idesc_mx4(UMMA_M, n, 0), idesc1 = idesc_mx4(UMMA_M, n, 1);
            const int acc = it % L::ACCS;
            if (!mbar_wait_warp(acc_empty(acc), ((it / L::ACCS) & 1) ^ 1)) {
                timed_out = true;
                break;
            }
            const uint32_t d = tmem_base + acc * NT;
            int left = p.K;
            for (int kb = 0; kb < kblocks; ++kb, left -= BK) {
                if (!mbar_wait_warp(full(slot), phase)) {
                    timed_out = true;
                    break;
                }
                tc_fence_after();
                // (every stage has its own columns: a copy into them comes behind the barrier that says that the
                // instructions which read them last are done)
                const uint32_t sf = tmem_base + L::SF_AT + slot * L::SF_STAGE_COLS;
                const uint64_t a = first + slot * (L::STAGE >> 4), scales = first_sf + slot * (L::STAGE >> 4);
                if (elect_one()) {
                    copy_scales<false, L::B_TILES>(sf, sf + SF_COLS, scales, scales + (SF_STAGE >> 4));
                    multiply_stage<false, L::B_TILES>(d, a, a + (L::A_BYTES >> 4), idesc0, idesc1, sf, sf + SF_COLS + u.sf_row / 32,
                                                      kb > 0, left >= BK ? 4 : (left + 63) / 64);
                    umma_commit(empty(slot));
                }
                __syncwarp();
                if (++slot == L::STAGES) slot = 0, phase ^= 1;
            }
            if (elect_one()) umma_commit(acc_full(acc));
            __syncwarp();
        }
    } else {
        // -------------------------------------------------------------------- epilogue
        const int q = warp & 3, half = (warp - 2) >> 2;
        int it = 0;
        for (int i = blockIdx.x; i < units; i += gridDim.x, ++it) {
            const Unit u = unit_of<NT, GROUPED>(p, i, m_tiles, start);
            const int acc = it % L::ACCS;
            constexpr int RUNS = NT / 16 / 2;
            const Rows<RUNS> r = rows_of<GROUPED, RUNS>(p, u, half, 2, lane);
            if (!mbar_wait_warp(acc_full(acc), (it / L::ACCS) & 1)) {
                timed_out = true;
                break;
            }
            tc_fence_after();
            const uint32_t d = tmem_base + acc * NT;
            if (p.out_type == MLS_BF16) store_unit<__nv_bfloat16, GROUPED, RUNS>(p, u, r, d, q, half, 2, lane);
            else store_unit<float, GROUPED, RUNS>(p, u, r, d, q, half, 2, lane);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty(acc));
        }
    }
    if (timed_out && p.status) atomicOr(p.status, MLS_STATUS_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, L::COLS);
}
}  // namespace mls_mx4
