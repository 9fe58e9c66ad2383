// Rows to 4-bit microscaled floating point and back.
//
// A block of 32 values with the largest magnitude m has the scale 2^max(floor(log2 m) - 2, -127); a value v becomes
// the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times the scale (a tie goes to the even code, what is larger to 6).  floor(log2 m)
// is m's exponent field, so the scale's byte is max(field - 2, 0), and dividing by the scale is an exact product with a
// power of two.  Bits of magnitudes order like the numbers, infinities and NaN above all others: the largest of them
// says both the scale and whether the block is a number at all (if not its scale is 255 and its codes are 0).
//
// Eight values a thread, four threads a block, a warp 256 of a row: 16 or 32 bytes a load, 4 bytes of codes a store,
// and the four scales of 128 values as one word.  What bounds it: the rows are read once and a quarter (or an eighth) of
// that is written.
#include "mx4.h"

namespace {
using namespace mls_mx4;

// Where a row comes from and where its scales go.
struct RowMap {
    int rows_per_mat, pairs;                       // plain rows: matrices of so many rows, or pairs of them
    const int *order, *idx, *offsets;              // sorted slots of a routed step (offsets == nullptr: plain rows)
    int top, n_experts, gather;                    // gather: row p is a copy of row order[p] / top
};

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int k0, int K, uint32_t (&bits)[8]) {
    if constexpr (sizeof(T) == 2) {
        if (VEC && k0 + 8 <= K) {
            const uint4 v = *reinterpret_cast<const uint4*>(row + k0);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bits[2 * i] = w[i] << 16;
                bits[2 * i + 1] = w[i] & 0xffff0000u;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            bits[i] = k0 + i < K ? (uint32_t)__bfloat16_as_ushort(row[k0 + i]) << 16 : 0u;
    } else {
        if (VEC && k0 + 8 <= K) {
            const uint4 a = *reinterpret_cast<const uint4*>(row + k0);
            const uint4 b = *reinterpret_cast<const uint4*>(row + k0 + 4);
            bits[0] = a.x, bits[1] = a.y, bits[2] = a.z, bits[3] = a.w;
            bits[4] = b.x, bits[5] = b.y, bits[6] = b.z, bits[7] = b.w;
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) bits[i] = k0 + i < K ? __float_as_uint(row[k0 + i]) : 0u;
    }
}

// Eight values in [-8, 8] as eight codes, the first in the lowest bits.
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

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
mx4_quantize_kernel(const T* __restrict__ x, long long ld, long long rows, int K, const RowMap map,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    chain_release();
    chain_wait();
    const int atoms = atoms_of(K), groups = atoms * 16, pitch = pitch_of(K);   // groups of 8: whole warps
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long p = i / groups;
    if (p >= rows) return;
    const int g = (int)(i - p * groups), k0 = g * 8;
    long long from = p;
    Place to;
    if (map.offsets) {
        const int slot = map.order[p], e = map.idx[slot];
        if (e >= map.n_experts) return;             // a slot of an output without weights: nobody reads it
        const int o = map.offsets[e], at = (int)p - o;
        if (map.gather) from = slot / map.top;
        to = {p, first_tile(o, e) + at / TILE_ROWS, at % TILE_ROWS};
    } else {
        to = place_of(p, map.rows_per_mat, map.pairs);
    }
    uint32_t bits[8];
    load8<T, VEC>(x + from * ld, k0, K, bits);
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, bits[j] & 0x7fffffffu);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const uint32_t field = most >> 23;
    const bool number = field < 255;
    const uint32_t scale = number ? (field > 2 ? field - 2 : 0) : 255;
    const float inverse = __uint_as_float((254 - (number ? scale : 0)) << 23);       // 2^(127 - scale)
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = number ? __uint_as_float(bits[j]) * inverse : 0.f;
    if (k0 < 2 * pitch) *reinterpret_cast<uint32_t*>(codes + to.row * pitch + g * 4) = pack8(v);
    const int lane = threadIdx.x & 31;
    uint32_t word = scale << (8 * ((lane >> 2) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if ((lane & 15) == 0)
        *reinterpret_cast<uint32_t*>(scales + (to.tile * atoms + (g >> 4)) * ATOM + row_in_atom(to.r)) = word;
}

// What codes and scales stand for; eight values a thread.
template <typename T>
__global__ void __launch_bounds__(256)
mx4_values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, long long rows, int K,
                  int rows_per_mat, int pairs, T* __restrict__ out, bool vec) {
    chain_release();
    chain_wait();
    const int pitch = pitch_of(K), groups = pitch / 4, atoms = atoms_of(K);
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long p = i / groups;
    if (p >= rows) return;
    const int g = (int)(i - p * groups), k0 = g * 8;
    if (k0 >= K) return;
    const Place at = place_of(p, rows_per_mat, pairs);
    const uint32_t scale = scales[(at.tile * atoms + (g >> 4)) * ATOM + row_in_atom(at.r) + ((g >> 2) & 3)];
    const uint32_t word = *reinterpret_cast<const uint32_t*>(codes + at.row * pitch + g * 4);
    // (2^(scale - 127); below 2^-126 the power has no exponent field of its own)
    const float power = scale == 255 ? __uint_as_float(0x7fffffffu)
                                     : __uint_as_float(scale ? scale << 23 : 0x00400000u);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t c = (word >> (4 * j)) & 15, low = c & 7;
        // 0, 0.5, 1, 1.5, 2, 3, 4, 6
        const float mag = low < 4 ? 0.5f * (float)low : (float)((2 + (low & 1)) << ((low - 4) >> 1));
        v[j] = (c & 8 ? -mag : mag) * power;
    }
    T* dst = out + p * K + k0;
    if (vec) {                                       // K is a multiple of 8 and the rows are aligned
        if constexpr (sizeof(T) == 2) {
            uint4 w;
            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
            for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);   // exact
            *reinterpret_cast<uint4*>(dst) = w;
        } else {
            *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (k0 + j < K) Elem<T>::store(dst + j, v[j]);
    }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
constexpr long long MOST_BLOCKS = 0x7fffffffLL;

template <typename T>
int quantize(const void* x, long long ld, long long rows, int K, const RowMap& map, uint8_t* codes, uint8_t* scales,
             cudaStream_t stream) {
    const long long blocks = (rows * (atoms_of(K) * 16LL) + 255) / 256;
    if (blocks > MOST_BLOCKS) return MLS_ERR_UNSUPPORTED;
    if (aligned16(x) && ld % (16 / (int)sizeof(T)) == 0)
        MLS_LAUNCH((mx4_quantize_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)x, ld, rows, K,
                   map, codes, scales);
    else
        MLS_LAUNCH((mx4_quantize_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)x, ld, rows, K,
                   map, codes, scales);
    return launch_status();
}
}  // namespace

// Plain rows (offsets == nullptr) of matrices of rows_per_mat rows each (pairs: gate and up in turn, interleaved), or the
// sorted slots of a routed step.
MLS_API int mls_mx4_quantize(const void* x, int dtype, long long ld, long long rows, int K, int rows_per_mat, int pairs,
                             const int* order, const int* idx, const int* offsets, int top, int n_experts, int gather,
                             void* codes, void* scales, void* stream) {
    if (rows <= 0) return 0;
    if (K <= 0 || rows_per_mat <= 0) return MLS_ERR_UNSUPPORTED;
    const RowMap map{rows_per_mat, pairs, order, idx, offsets, top, n_experts, gather};
    return dtype == MLS_BF16
               ? quantize<__nv_bfloat16>(x, ld, rows, K, map, (uint8_t*)codes, (uint8_t*)scales, (cudaStream_t)stream)
               : quantize<float>(x, ld, rows, K, map, (uint8_t*)codes, (uint8_t*)scales, (cudaStream_t)stream);
}

MLS_API int mls_mx4_values(const void* codes, const void* scales, long long rows, int K, int rows_per_mat, int pairs,
                           void* out, int dtype, void* stream) {
    if (rows <= 0) return 0;
    if (K <= 0 || rows_per_mat <= 0) return MLS_ERR_UNSUPPORTED;
    const long long blocks = (rows * (pitch_of(K) / 4) + 255) / 256;
    if (blocks > MOST_BLOCKS) return MLS_ERR_UNSUPPORTED;
    const bool vec = K % 8 == 0 && aligned16(out);
    if (dtype == MLS_BF16)
        MLS_LAUNCH((mx4_values_kernel<__nv_bfloat16>), dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream,
                   (const uint8_t*)codes, (const uint8_t*)scales, rows, K, rows_per_mat, pairs, (__nv_bfloat16*)out, vec);
    else
        MLS_LAUNCH((mx4_values_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream,
                   (const uint8_t*)codes, (const uint8_t*)scales, rows, K, rows_per_mat, pairs, (float*)out, vec);
    return launch_status();
}
