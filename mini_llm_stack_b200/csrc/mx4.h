// 4-bit microscaled floating point: where codes and scales lie.
//
// A row of K values is cut into blocks of 32.  Codes: two to a byte, the even place in the low bits, a row's
// blocks one after another (16 bytes each), rows `pitch_of(K)` bytes apart.  Scales: one byte a block, the biased
// exponent of a power of two (255: the block is no number).  The scales of 128 rows x 128 of K form an atom of 512
// bytes in the order in which they enter tensor memory: row r's four bytes at (r % 32) * 16 + (r / 32) * 4.  A
// matrix is cut into tiles of 128 rows, and a tile's atoms follow one another along K, an even number of them (a
// product takes two at a time).
#pragma once
#include "common.cuh"
#include <atomic>
#include <cuda_fp16.h>
#include <string.h>

namespace mls_mx4 {
constexpr int BLOCK = 32;
constexpr int TILE_ROWS = 128;
constexpr int ATOM = 512;

__host__ __device__ constexpr int pitch_of(int K) { return (K + BLOCK - 1) / BLOCK * (BLOCK / 2); }
__host__ __device__ constexpr int atoms_of(int K) { return 2 * ((K + 255) / 256); }
// Bytes from a tile's first atom to a row's four scales in its atom.
__host__ __device__ constexpr unsigned row_in_atom(unsigned r) { return (r & 31) * 16 + ((r >> 5) & 3) * 4; }

// Rows of the pairs [2, N, K] of gate and up matrices lie interleaved, 16 of the gate's and 16 of up's in turn (N filled up
// to a multiple of 16): an output's two sums are then 16 lanes of a warp apart.
__host__ __device__ constexpr int pair_rows(int N) { return (N + 15) / 16 * 32; }
__host__ __device__ constexpr int pair_row(int which, int n) { return n / 16 * 32 + which * 16 + n % 16; }

// Where row p of matrices of N rows each lies: its row of codes, the tile of its scales and its row in that.
struct Place {
    unsigned row, tile, r;
};
__device__ __forceinline__ Place place_of(unsigned p, unsigned N, bool pairs) {
    if (p < N && !pairs) return {p, p / TILE_ROWS, p % TILE_ROWS};
    const unsigned mat = p / N, n = p - mat * N;
    const unsigned rows = pairs ? pair_rows((int)N) : N, at = pairs ? pair_row((int)(mat & 1), (int)n) : n;
    const unsigned m = pairs ? mat >> 1 : mat;
    return {m * rows + at, m * ((rows + TILE_ROWS - 1) / TILE_ROWS) + at / TILE_ROWS, at % TILE_ROWS};
}

// The sorted rows of a routed step: an expert's rows begin with a tile of their own.  Expert e's first tile is
// offsets[e] / 128 + e: with c rows behind offset o it takes ceil(c / 128) tiles, and (o + c) / 128 + 1 - o / 128,
// the distance to the next expert's, is never less.
__device__ __forceinline__ int first_tile(int offset, int e) { return offset / TILE_ROWS + e; }

// Where a row that is quantised comes from and where its scales go.
struct RowMap {
    int rows_per_mat, pairs;                       // plain rows: matrices of so many rows, or pairs of them
    const int *order, *idx, *offsets;              // sorted slots of a routed step (offsets == nullptr: plain rows)
    int top, n_experts, gather;                    // gather: row p is a copy of row order[p] / top
};
// What a C entry does, with an exception's end as an error code.
template <typename Body>
static inline int guarded(Body body) {
    try {
        return body();
    } catch (...) {
        return (int)cudaErrorMemoryAllocation;
    }
}

// A kernel's limit of shared memory, set once on every device.
class SharedLimit {
public:
    template <typename Kernel>
    int set(Kernel kernel, int bytes) {
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e != cudaSuccess) return (int)e;
        const unsigned long long bit = 1ull << (device & 63);
        if (device < 64 && (done_.load() & bit)) return 0;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) done_.fetch_or(bit);
        return (int)e;
    }

private:
    std::atomic<unsigned long long> done_{0};
};

// A launch that starts when the kernels before it have finished.
template <typename... Params, typename... Args>
static inline int launch_plain(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                               Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    return (int)cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// Rows [rows, K] of float32 or bfloat16, ld values apart, into codes and scales.
int quantize_rows(const void* x, int dtype, long long ld, long long rows, int K, const RowMap& map, uint8_t* codes,
                  uint8_t* scales, bool chained, cudaStream_t stream);
// The tokens' rows [tokens, K] once each, into all of their sorted slots; places: 8 bytes a slot of scratch.
int quantize_tokens(const void* x, int dtype, long long ld, long long tokens, int K, const RowMap& map, long long slots,
                    void* places, uint8_t* codes, uint8_t* scales, cudaStream_t stream);

// Eight neighbouring values of a row as they lie (zeros behind the row's end).
template <typename T>
struct Eight {
    uint32_t w[2 * sizeof(T)];
};
// 8 EIGHTS of them as the 16-byte pieces of memory that they lie in, asked for by load_raw and put into place by settle, so that a
// thread's loads are under way together.  VEC: rows begin at 16-byte places, the values' pieces are theirs alone; else neighbours
// are read along, of the same matrix (its ends, which may lie within a piece, value by value).
template <typename T, bool VEC, int EIGHTS>
struct Raw {
    static constexpr int OWN = EIGHTS * 8 * sizeof(T) / 16, PIECES = OWN + !VEC;
    uint4 piece[PIECES];
};
template <typename T, bool VEC, int EIGHTS>
__device__ __forceinline__ void load_raw(const T* matrix, const T* end, const T* row, int k0, int K, Raw<T, VEC, EIGHTS>& r) {
    if constexpr (VEC) {
#pragma unroll
        for (int e = 0; e < EIGHTS; ++e) {
            const int k = k0 + 8 * e;
            uint32_t w[2 * sizeof(T)];
            if (k + 8 <= K) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                    const uint4 u = reinterpret_cast<const uint4*>(row + k)[i];
                    w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
                }
            } else if constexpr (sizeof(T) == 2) {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = (k + 2 * i < K ? (uint32_t)h[k + 2 * i] : 0u) |
                           (k + 2 * i + 1 < K ? (uint32_t)h[k + 2 * i + 1] << 16 : 0u);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = k + i < K ? __float_as_uint(row[k + i]) : 0u;
            }
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                r.piece[e * (sizeof(T) / 2) + i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
        return;
    }
    const uintptr_t lo = reinterpret_cast<uintptr_t>(matrix), hi = reinterpret_cast<uintptr_t>(end);
    const uintptr_t from = reinterpret_cast<uintptr_t>(row + k0) & ~(uintptr_t)15, behind = reinterpret_cast<uintptr_t>(row + K);
#pragma unroll
    for (int i = 0; i < Raw<T, VEC, EIGHTS>::PIECES; ++i) {
        const uintptr_t at = from + 16 * i;
        r.piece[i] = make_uint4(0, 0, 0, 0);
        if (k0 >= K || at >= behind) continue;
        if (at >= lo && at + 16 <= hi) {
            r.piece[i] = *reinterpret_cast<const uint4*>(at);
        } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < 16 / (int)sizeof(T); ++x) {
                const uintptr_t one = at + x * sizeof(T);
                if (one < lo || one >= hi) continue;
                if constexpr (sizeof(T) == 2) w[x / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(one) << (x % 2 * 16);
                else w[x] = *reinterpret_cast<const uint32_t*>(one);
            }
            r.piece[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}
template <typename T, bool VEC, int EIGHTS>
__device__ __forceinline__ void settle(const Raw<T, VEC, EIGHTS>& r, const T* row, int k0, int K, Eight<T> (&v)[EIGHTS]) {
    constexpr int WORDS = 4 * Raw<T, VEC, EIGHTS>::OWN, ALL = 4 * Raw<T, VEC, EIGHTS>::PIECES, PER = 4 / sizeof(T);
    uint32_t w[ALL];
#pragma unroll
    for (int i = 0; i < ALL / 4; ++i)
        w[4 * i] = r.piece[i].x, w[4 * i + 1] = r.piece[i].y, w[4 * i + 2] = r.piece[i].z, w[4 * i + 3] = r.piece[i].w;
    if (!VEC) {
        const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(row + k0) & 15);
#pragma unroll
        for (int i = 0; i + 1 < ALL; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
#pragma unroll
        for (int i = 0; i + 2 < ALL; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
        if (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = off & 2 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
        }
    }
    if (!VEC && k0 + 8 * EIGHTS > K) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            if (k0 + i * PER >= K) w[i] = 0;
            else if (PER == 2 && k0 + i * PER + 1 >= K) w[i] &= 0xffffu;
        }
    }
#pragma unroll
    for (int i = 0; i < WORDS; ++i) v[i / (2 * sizeof(T))].w[i % (2 * sizeof(T))] = w[i];
}

// Values in [-8, 8] as codes, the first in the lowest bits.
__device__ __forceinline__ uint32_t pack8(const float (&v)[8]) {
    uint32_t out;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(out)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return out;
}
// And back: two values of a byte.
__device__ __forceinline__ float2 unpack2(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h) : "r"(byte));
    __half2 two;
    memcpy(&two, &h, 4);
    return __half22float2(two);
}
// The largest magnitude of three; NaN where one is none.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
    float m;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}

// A lane's 8 EIGHTS neighbouring values as codes; 4 / EIGHTS lanes share a block.  `scales` is, in every (16 / EIGHTS)th lane, the
// four scales of the 128 values from that lane's on.
//
// A block of 32 values with the largest magnitude m has the scale 2^max(floor(log2 m) - 2, -127); a value v becomes
// the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times the scale (a tie goes to the even code, what is larger to 6).  floor(log2 m)
// is m's exponent field, so the scale's byte is max(field - 2, 0), and dividing by the scale is an exact product with a
// power of two.  The bits of the largest magnitude say both the scale and, as infinities and NaN have the largest exponent
// field, whether the block is a number at all (if not its scale is 255, whatever its codes).
template <typename T, int EIGHTS>
__device__ __forceinline__ void quantize_lane(const Eight<T> (&x)[EIGHTS], int lane, uint32_t (&codes)[EIGHTS], uint32_t& scales) {
    float v[EIGHTS][8], largest = 0.f;
#pragma unroll
    for (int i = 0; i < EIGHTS; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t bits;
            if constexpr (sizeof(T) == 2) bits = j & 1 ? x[i].w[j / 2] & 0xffff0000u : x[i].w[j / 2] << 16;
            else bits = x[i].w[j];
            v[i][j] = __uint_as_float(bits);
        }
#pragma unroll
        for (int j = 0; j < 8; j += 2) largest = max_abs(largest, v[i][j], v[i][j + 1]);
    }
    uint32_t most = __float_as_uint(largest);
#pragma unroll
    for (int o = 1; o < 4 / EIGHTS; o *= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    const uint32_t field = most >> 23;
    const uint32_t scale = field == 255 ? 255 : max(field, 2u) - 2;
    const float inverse = __uint_as_float((254 - min(scale, 253u)) << 23);           // 2^(127 - scale)
#pragma unroll
    for (int i = 0; i < EIGHTS; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= inverse;
        codes[i] = pack8(v[i]);
    }
    scales = scale << (8 * ((lane * EIGHTS >> 2) & 3));
    scales |= __shfl_xor_sync(0xffffffffu, scales, 4 / EIGHTS);
    scales |= __shfl_xor_sync(0xffffffffu, scales, 8 / EIGHTS);
}
}  // namespace mls_mx4
