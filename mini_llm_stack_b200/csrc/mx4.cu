// Rows to 4-bit microscaled floating point (mx4.h) and back.
//
// Sixteen values a thread, two threads a block, a warp 512 of a row: 8 bytes of codes a store, the four scales of 128 values
// as one word (eight values a thread: 33.9 us for 14,336 x 4,096 bfloat16 values instead of 25.3, most of it what a task
// costs beside its values).  What bounds it: the rows are read once and a quarter (or an eighth) of that is written; 14,336 x
// 4,096 float32 values in 39.5 us (6.7 TB/s), bfloat16 in 25.3 (5.9 TB/s, the instructions beside the loads).  Back to
// float32 43.3 us, to bfloat16 26.3.
#include "mx4.h"
#include <type_traits>

namespace {
using namespace mls_mx4;

// A warp's task: PART values of a row.  Tasks are numbered along the rows; a warp takes UNROLL of them, as many apart as there
// are warps, whose loads are under way together.
constexpr int UNROLL = 4, PART_VALUES = 256;                       // of values read back
constexpr int QUANTIZE_UNROLL = 2, QUANTIZE_PART = 512;           // of values quantised
constexpr int RESIDENT = 3;                                       // blocks that fit an SM, at least
struct Tasks {
    unsigned rows, chunks, step_row, step_chunk;
    // All blocks are resident at once (RESIDENT an SM).  Only then does a kernel let its successors start early: one with tensor
    // memory, a whole SM a block and blocks that wait for one another shall not become resident SM by SM while the last round of
    // many drains (a pair's product behind such a quantisation did not end under a profiler, for a reason that reading did not
    // show).  It costs nothing: 14,336 x 4,096 float32 values there and back in 87.3 us, 88.1 with early starts.
    bool at_once;
    __device__ __forceinline__ void next(unsigned& row, unsigned& chunk) const {
        row += step_row, chunk += step_chunk;
        if (chunk >= chunks) chunk -= chunks, ++row;
    }
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(256, RESIDENT)
mx4_quantize_kernel(const T* __restrict__ x, const T* end, long long ld, const Tasks tasks, int K, const RowMap map,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    if (tasks.at_once) chain_release();
    chain_wait();
    const int pitch = pitch_of(K), atoms = atoms_of(K), lane = threadIdx.x & 31;
    const unsigned first = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    unsigned p = first / tasks.chunks, chunk = first - p * tasks.chunks;
    Raw<T, VEC, 2> raw[QUANTIZE_UNROLL];
    const T* from[QUANTIZE_UNROLL];
    unsigned row[QUANTIZE_UNROLL], at[QUANTIZE_UNROLL];
    int slot[QUANTIZE_UNROLL], e[QUANTIZE_UNROLL], o[QUANTIZE_UNROLL];
    // (a slot's number, its expert and that one's first row: loads that wait for one another, but for no other task's)
    if (map.offsets) {
        unsigned p1 = p, c1 = chunk;
#pragma unroll
        for (int j = 0; j < QUANTIZE_UNROLL; ++j) {
            row[j] = p1;
            slot[j] = p1 < tasks.rows ? map.order[p1] : 0;
            tasks.next(p1, c1);
        }
#pragma unroll
        for (int j = 0; j < QUANTIZE_UNROLL; ++j) e[j] = row[j] < tasks.rows ? map.idx[slot[j]] : 0;
#pragma unroll
        for (int j = 0; j < QUANTIZE_UNROLL; ++j) o[j] = row[j] < tasks.rows && e[j] < map.n_experts ? map.offsets[e[j]] : 0;
    }
#pragma unroll
    for (int j = 0; j < QUANTIZE_UNROLL; ++j) {
        row[j] = p, at[j] = chunk;
        if (p < tasks.rows) {
            from[j] = x + (long long)(map.gather ? (unsigned)(slot[j] / map.top) : p) * ld;
            load_raw(x, end, from[j], (int)chunk * QUANTIZE_PART + lane * 16, K, raw[j]);
        }
        tasks.next(p, chunk);
    }
#pragma unroll
    for (int j = 0; j < QUANTIZE_UNROLL; ++j) {
        if (row[j] >= tasks.rows) break;
        Eight<T> held[2];
        settle(raw[j], from[j], (int)at[j] * QUANTIZE_PART + lane * 16, K, held);
        uint32_t word, packed[2];
        quantize_lane(held, lane, packed, word);
        Place to;
        if (map.offsets) {
            if (e[j] >= map.n_experts) continue;    // a slot of an output without weights: nobody reads it
            const unsigned r = row[j] - o[j];
            to = {row[j], first_tile(o[j], e[j]) + r / TILE_ROWS, r % TILE_ROWS};
        } else {
            to = place_of(row[j], map.rows_per_mat, map.pairs);
        }
        const int byte = (int)at[j] * (QUANTIZE_PART / 2) + lane * 8, atom = (int)at[j] * 4 + (lane >> 3);
        if (byte < pitch)
            *reinterpret_cast<uint2*>(codes + (size_t)to.row * pitch + byte) = make_uint2(packed[0], packed[1]);
        if ((lane & 7) == 0 && atom < atoms)
            *reinterpret_cast<uint32_t*>(scales + ((size_t)to.tile * atoms + atom) * ATOM + row_in_atom(to.r)) = word;
    }
}

// Where the slots of a routed step lie among its sorted rows: the row of codes, and that of scales counted in tiles of 128.
__global__ void __launch_bounds__(256)
mx4_places_kernel(const RowMap map, int slots, int2* __restrict__ places) {
    const int p = blockIdx.x * blockDim.x + threadIdx.x;
    if (p >= slots) return;
    const int slot = map.order[p], e = map.idx[slot];
    int2 place = {-1, 0};                            // (a slot of an output without weights: nobody reads it)
    if (e < map.n_experts) {
        const int o = map.offsets[e];
        place = {p, first_tile(o, e) * TILE_ROWS + p - o};
    }
    places[slot] = place;
}

// A token is quantised once and stored to all of its slots: a warp's task is 512 values of a token.  What bounds it is what L2 takes
// in, 27 MB for 12,288 slots of 4,096, the scales among them in words of four bytes: 11.5 us and 2.9 for the places (the tokens'
// codes and scales as rows of their own, copied to the slots by a second kernel: 17).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
mx4_tokens_kernel(const T* __restrict__ x, const T* end, long long ld, const Tasks tasks, int K, int top, int slots, int tiles,
                  const int2* __restrict__ places, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int pitch = pitch_of(K), atoms = atoms_of(K), lane = threadIdx.x & 31;
    const unsigned first = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    unsigned token = first / tasks.chunks, chunk = first - token * tasks.chunks;
    for (; token < tasks.rows; tasks.next(token, chunk)) {
        const int k0 = (int)chunk * QUANTIZE_PART + lane * 16;
        const T* row = x + (long long)token * ld;
        Raw<T, VEC, 2> raw;
        load_raw(x, end, row, k0, K, raw);
        const int byte = (int)chunk * (QUANTIZE_PART / 2) + lane * 8, atom = (int)chunk * 4 + (lane >> 3);
        uint32_t word = 0, packed[2];
        for (int j0 = 0; j0 < top; j0 += 32) {
            const int2 mine = j0 + lane < top ? places[(size_t)token * top + j0 + lane] : make_int2(-1, 0);
            if (j0 == 0) {
                Eight<T> held[2];
                settle(raw, row, k0, K, held);
                quantize_lane(held, lane, packed, word);
            }
            const int n = min(32, top - j0);
            for (int j = 0; j < n; ++j) {
                const int to = __shfl_sync(0xffffffffu, mine.x, j), at = __shfl_sync(0xffffffffu, mine.y, j);
                // (a place that the routing's arrays left out is none)
                if ((unsigned)to >= (unsigned)slots || (unsigned)at >= (unsigned)tiles * TILE_ROWS) continue;
                if (byte < pitch)
                    *reinterpret_cast<uint2*>(codes + (size_t)to * pitch + byte) = make_uint2(packed[0], packed[1]);
                if ((lane & 7) == 0 && atom < atoms)
                    *reinterpret_cast<uint32_t*>(scales + ((size_t)(at / TILE_ROWS) * atoms + atom) * ATOM +
                                                 row_in_atom(at % TILE_ROWS)) = word;
            }
        }
    }
}

// What codes and scales stand for, in the same tasks.  A lane takes PER neighbouring values, 16 bytes of output, once in 256
// bfloat16 values and twice in 256 of float32 (two stores of 16 bytes a lane, 32 apart from the next lane's: 62 us for
// 14,336 x 4,096 instead of 43).  Without VEC rows begin anywhere.  A lane then stores float32 values one by one; of bfloat16 it takes
// the values of a 16-byte piece of the output, whose codes may lie in two words and two blocks, and only the pieces at a row's
// ends are stored so (10,000 x 3,999: 34 us instead of 118).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256, 2 * RESIDENT)
mx4_values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const Tasks tasks, int K,
                  int rows_per_mat, int pairs, T* __restrict__ out) {
    if (tasks.at_once) chain_release();
    chain_wait();
    constexpr int PER = 16 / sizeof(T), TIMES = 8 / PER;
    constexpr bool PIECES = !VEC && PER == 8;
    using Word = typename std::conditional<PER == 8, uint32_t, uint16_t>::type;      // PER codes
    const int pitch = pitch_of(K), lane = threadIdx.x & 31;
    const unsigned first = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    unsigned p = first / tasks.chunks, chunk = first - p * tasks.chunks;
    uint32_t words[UNROLL][TIMES], scale[UNROLL][TIMES], scale_behind[UNROLL];
    unsigned row[UNROLL], chunk_of[UNROLL];
    // a lane's first value in a task (PIECES: of a piece that may begin before the row)
    auto value = [&](unsigned row, unsigned chunk, int h) {
        const unsigned before = PIECES ? ((unsigned)(reinterpret_cast<uintptr_t>(out) / sizeof(T)) + row * (unsigned)K) % PER : 0;
        return (int)(chunk * 256 + (h * 32 + lane) * PER) - (int)before;
    };
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
        row[j] = p, chunk_of[j] = chunk;
        if (p < tasks.rows) {
            const Place at = place_of(p, rows_per_mat, pairs);
            const uint8_t* row_codes = codes + (size_t)at.row * pitch;
            if constexpr (PIECES) {
                const uint8_t* row_scales = scales + (size_t)at.tile * atoms_of(K) * ATOM + row_in_atom(at.r);
                const int k = value(p, chunk, 0), byte = (k >> 3) * 4;
                const unsigned k1 = max(k, 0), k2 = min(k + PER - 1, K - 1);
                uint32_t a = 0, b = 0;
                if (byte >= 0 && byte < pitch) a = *reinterpret_cast<const uint32_t*>(row_codes + byte);
                if (byte + 4 < pitch) b = *reinterpret_cast<const uint32_t*>(row_codes + byte + 4);
                words[j][0] = __funnelshift_r(a, b, 4 * (k & 7));
                scale[j][0] = k < K ? row_scales[(k1 >> 7) * ATOM + (k1 >> 5 & 3)] : 0;
                scale_behind[j] = k < K ? row_scales[(k2 >> 7) * ATOM + (k2 >> 5 & 3)] : 0;
            } else {
                const uint8_t* task_scales = scales + ((size_t)at.tile * tasks.chunks + chunk) * (2 * ATOM) + row_in_atom(at.r);
#pragma unroll
                for (int h = 0; h < TIMES; ++h) {
                    const int k = (h * 32 + lane) * PER, byte = (int)chunk * 128 + k / 2;          // in the task
                    words[j][h] = byte < pitch ? *reinterpret_cast<const Word*>(row_codes + byte) : 0;
                    scale[j][h] = task_scales[k / 128 * ATOM + k / 32 % 4];
                }
            }
        }
        tasks.next(p, chunk);
    }
    // (2^(scale - 127); below 2^-126 the power has no exponent field of its own)
    auto power_of = [](uint32_t c) { return __uint_as_float(c == 255 ? 0x7fffffffu : c ? c << 23 : 0x00400000u); };
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
        if (row[j] >= tasks.rows) break;
#pragma unroll
        for (int h = 0; h < TIMES; ++h) {
            const int k0 = value(row[j], chunk_of[j], h);
            if (k0 >= K) continue;
            const float power = power_of(scale[j][h]), behind = PIECES ? power_of(scale_behind[j]) : power;
            const int left = 32 - (k0 & 31);                       // values to the next block
            float v[PER];
#pragma unroll
            for (int i = 0; i < PER / 2; ++i) {
                const float2 f = unpack2(words[j][h] >> (8 * i));
                v[2 * i] = f.x * (2 * i < left ? power : behind), v[2 * i + 1] = f.y * (2 * i + 1 < left ? power : behind);
            }
            T* dst = out + (size_t)row[j] * K + k0;
            if (VEC || (PIECES && k0 >= 0 && k0 + PER <= K)) {
                if constexpr (PER == 8) {
                    uint4 w;
                    __nv_bfloat162* b = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) b[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);   // exact
                    *reinterpret_cast<uint4*>(dst) = w;
                } else {
                    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (k0 + i >= 0 && k0 + i < K) Elem<T>::store(dst + i, v[i]);
            }
        }
    }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
// The tasks and the blocks of eight warps for them; false: more tasks than a launch numbers.
bool tasks_of(long long rows, int K, int part, int unroll, Tasks& tasks, unsigned& blocks) {
    const long long chunks = (K + part - 1) / part, n = rows * chunks;
    if (n > 0x7fffffffLL) return false;
    blocks = (unsigned)((n + 8 * unroll - 1) / (8 * unroll));
    // (few tasks: a warp each, as long as the SMs have room for them)
    const unsigned room = 4u * (unsigned)sm_count(), each = (unsigned)((n + 7) / 8);
    if (blocks < room) blocks = each < room ? each : room;
    const unsigned warps = 8 * blocks;
    tasks = {(unsigned)rows, (unsigned)chunks, warps / (unsigned)chunks, warps % (unsigned)chunks,
             blocks <= RESIDENT * (unsigned)sm_count()};
    return true;
}

template <typename T>
int quantize(const void* x, long long ld, long long rows, int K, const RowMap& map, uint8_t* codes, uint8_t* scales,
             bool chained, cudaStream_t stream) {
    Tasks tasks;
    unsigned blocks;
    if (!tasks_of(rows, K, QUANTIZE_PART, QUANTIZE_UNROLL, tasks, blocks)) return MLS_ERR_UNSUPPORTED;
    auto* kernel = aligned16(x) && ld % (16 / (int)sizeof(T)) == 0 ? mx4_quantize_kernel<T, true> : mx4_quantize_kernel<T, false>;
    const T *first = (const T*)x, *end = first + ((map.gather ? rows / map.top : rows) - 1) * ld + K;
    const int rc = chained ? launch_chained(kernel, dim3(blocks), dim3(256), 0, stream, first, end, ld, tasks, K, map, codes, scales)
                           : launch_plain(kernel, dim3(blocks), dim3(256), 0, stream, first, end, ld, tasks, K, map, codes, scales);
    return rc ? rc : launch_status();
}

template <typename T>
int tokens_to_slots(const void* x, long long ld, long long tokens, int K, const RowMap& map, long long slots, const int2* places,
                    uint8_t* codes, uint8_t* scales, cudaStream_t stream) {
    Tasks tasks;
    unsigned blocks;
    if (!tasks_of(tokens, K, QUANTIZE_PART, 1, tasks, blocks)) return MLS_ERR_UNSUPPORTED;
    auto* kernel = aligned16(x) && ld % (16 / (int)sizeof(T)) == 0 ? mx4_tokens_kernel<T, true> : mx4_tokens_kernel<T, false>;
    const T *first = (const T*)x, *end = first + (tokens - 1) * ld + K;
    const int rc = launch_plain(kernel, dim3(blocks), dim3(256), 0, stream, first, end, ld, tasks, K, map.top, (int)slots,
                                (int)(slots / TILE_ROWS + map.n_experts + 1), places, codes, scales);
    return rc ? rc : launch_status();
}
}  // namespace

namespace mls_mx4 {
int quantize_rows(const void* x, int dtype, long long ld, long long rows, int K, const RowMap& map, uint8_t* codes,
                  uint8_t* scales, bool chained, cudaStream_t stream) {
    return dtype == MLS_BF16 ? quantize<__nv_bfloat16>(x, ld, rows, K, map, codes, scales, chained, stream)
                             : quantize<float>(x, ld, rows, K, map, codes, scales, chained, stream);
}
int quantize_tokens(const void* x, int dtype, long long ld, long long tokens, int K, const RowMap& map, long long slots,
                    void* places, uint8_t* codes, uint8_t* scales, cudaStream_t stream) {
    const int rc = launch_plain(mx4_places_kernel, dim3((unsigned)((slots + 255) / 256)), dim3(256), 0, stream, map, (int)slots,
                                (int2*)places);
    if (rc) return rc;
    return dtype == MLS_BF16
               ? tokens_to_slots<__nv_bfloat16>(x, ld, tokens, K, map, slots, (const int2*)places, codes, scales, stream)
               : tokens_to_slots<float>(x, ld, tokens, K, map, slots, (const int2*)places, codes, scales, stream);
}
}  // namespace mls_mx4

// Matrices of rows_per_mat rows each (pairs: gate and up in turn, left interleaved).
MLS_API int mls_mx4_quantize(const void* x, int dtype, long long ld, long long rows, int K, int rows_per_mat, int pairs,
                             void* codes, void* scales, void* stream) {
    if (rows <= 0) return 0;
    if (K <= 0 || rows_per_mat <= 0) return MLS_ERR_UNSUPPORTED;
    const RowMap map{rows_per_mat, pairs, nullptr, nullptr, nullptr, 1, 0, 0};
    return quantize_rows(x, dtype, ld, rows, K, map, (uint8_t*)codes, (uint8_t*)scales, true, (cudaStream_t)stream);
}

MLS_API int mls_mx4_values(const void* codes, const void* scales, long long rows, int K, int rows_per_mat, int pairs,
                           void* out, int dtype, void* stream) {
    if (rows <= 0) return 0;
    if (K <= 0 || rows_per_mat <= 0) return MLS_ERR_UNSUPPORTED;
    Tasks tasks;
    unsigned blocks;
    const int per = dtype == MLS_BF16 ? 8 : 4;
    const bool vec = K % per == 0 && aligned16(out);
    // (bfloat16 rows that begin within a piece of 16 bytes may reach into one more)
    if (!tasks_of(rows, !vec && per == 8 ? K + per - 1 : K, PART_VALUES, UNROLL, tasks, blocks)) return MLS_ERR_UNSUPPORTED;
    const cudaStream_t s = (cudaStream_t)stream;
    const uint8_t *c = (const uint8_t*)codes, *f = (const uint8_t*)scales;
    const dim3 grid(blocks), block(256);
    if (dtype == MLS_BF16) {
        __nv_bfloat16* to = (__nv_bfloat16*)out;
        if (vec) MLS_LAUNCH((mx4_values_kernel<__nv_bfloat16, true>), grid, block, 0, s, c, f, tasks, K, rows_per_mat, pairs, to);
        else MLS_LAUNCH((mx4_values_kernel<__nv_bfloat16, false>), grid, block, 0, s, c, f, tasks, K, rows_per_mat, pairs, to);
    } else {
        float* to = (float*)out;
        if (vec) MLS_LAUNCH((mx4_values_kernel<float, true>), grid, block, 0, s, c, f, tasks, K, rows_per_mat, pairs, to);
        else MLS_LAUNCH((mx4_values_kernel<float, false>), grid, block, 0, s, c, f, tasks, K, rows_per_mat, pairs, to);
    }
    return launch_status();
}
