// Products of 4-bit microscaled rows and weights on the 5th-generation tensor cores: for one matrix, or expert by
// expert over the sorted slots p of a routed step (offsets[e] <= p < offsets[e + 1]),
//
//   DOWN    out[m, n] = W a_m                        W [N, K]; routed: float32 per_slot[order[p], n], times the slot's
//                                                    weight with `scale`
//   GATED   out[m, n] = unit(s Wg a_m, s Wu a_m)     W [2, N, K], interleaved (mx4.h); s: the slot's weight with `scale`,
//                                                    else 1
//   RELU2   out[m, n] = relu(s W a_m)^2              W [N, K]
//
// Values are e2m1, scales e8m0 for 32 of K: kind::mxf4 multiplies them exactly and adds up in float32, k ascending.  The
// weights take the 128-row side of the instruction, the rows the other one, up to NT at a time and rounded up to 16.
// A stage is 256 of K: 16 KB of weight codes and 1 KB of their scales, 128 bytes a row and 8 of its scales; codes come by TMA
// with the 128-byte swizzle, scales as they lie (mx4.h) and go on into tensor memory, in the order of the instructions.
//
// Warp roles: 0 = TMA producer, 1 = tensor memory and instructions, 2..9 = epilogue (two warps a quarter of the lanes,
// taking 16 columns in turn).  Every wait is bounded; one that runs out sets MLS_STATUS_TIMEOUT, and the kernel frees its
// tensor memory and returns.
#include "mx4_few.h"
#include "mx4_gemm.h"
#include "mx4_pair.h"
#include <map>
#include <mutex>
#include <tuple>

namespace {
using namespace mls_mx4;

template <int NT, bool GROUPED>
__global__ void __launch_bounds__(THREADS, 1)
mx4_product_kernel(const Product p, const __grid_constant__ CUtensorMap rows_map,
                   const __grid_constant__ CUtensorMap w_map) {
    product_block<NT, GROUPED>(p, &rows_map, &w_map);
}

template <int NT, bool GROUPED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairPlan<NT>::THREADS, 1)
mx4_pair_kernel(const Product p, const __grid_constant__ CUtensorMap rows_map, const __grid_constant__ CUtensorMap half_map,
                const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap sf_rows_map,
                const __grid_constant__ CUtensorMap sf_w_map) {
    pair_block<NT, GROUPED>(p, &rows_map, &half_map, &w_map, &sf_rows_map, &sf_w_map);
}

template <int NR, bool FUSED>
__global__ void __launch_bounds__(FEW_THREADS)
mx4_few_kernel(const FewProduct p, const __grid_constant__ CUtensorMap rows_map, const __grid_constant__ CUtensorMap w_map) {
    few_block<NR, FUSED>(p, &rows_map, &w_map);
}

// Tensor maps by what they describe, as the other products keep theirs.
struct MapKey {
    const void* ptr;
    long long rows;
    int k, box, kind;
    bool operator<(const MapKey& o) const {
        return std::tie(ptr, rows, k, box, kind) < std::tie(o.ptr, o.rows, o.k, o.box, o.kind);
    }
};
template <typename Encode>
bool kept_map(const MapKey& key, CUtensorMap* out, Encode encode) {
    static std::map<MapKey, CUtensorMap> maps;
    static std::mutex lock;
    std::lock_guard<std::mutex> guard(lock);
    auto it = maps.find(key);
    if (it == maps.end()) {
        if (maps.size() > 4096) maps.clear();
        EncodeTiledFn fn = encode_fn();
        CUtensorMap m;
        if (!fn || encode(fn, &m) != CUDA_SUCCESS) return false;
        it = maps.emplace(key, m).first;
    }
    *out = it->second;
    return true;
}
// Codes [rows, pitch] in boxes of box_rows x 128 bytes.
bool codes_map(const void* ptr, long long rows, int K, int box_rows, CUtensorMap* out) {
    return kept_map({ptr, rows, K, box_rows, 0}, out, [&](EncodeTiledFn fn, CUtensorMap* m) {
        const cuuint64_t size[2] = {(cuuint64_t)pitch_of(K), (cuuint64_t)rows}, stride[1] = {(cuuint64_t)pitch_of(K)};
        const cuuint32_t box[2] = {(cuuint32_t)CODE_ROW, (cuuint32_t)box_rows}, step[2] = {1, 1};
        return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), size, stride, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
}
// Scales [tiles, stages of K, 1,024 bytes] in boxes of the same stage of box_tiles tiles.
bool scales_map(const void* ptr, long long tiles, int K, int box_tiles, CUtensorMap* out) {
    return kept_map({ptr, tiles, K, box_tiles, 1}, out, [&](EncodeTiledFn fn, CUtensorMap* m) {
        const cuuint64_t stages = (K + BK - 1) / BK;
        const cuuint64_t size[3] = {SF_STAGE / 4, stages, (cuuint64_t)tiles}, stride[2] = {SF_STAGE, stages * SF_STAGE};
        const cuuint32_t box[3] = {SF_STAGE / 4, 1, (cuuint32_t)box_tiles}, step[3] = {1, 1, 1};
        return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(ptr), size, stride, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
}

// Products of many rows are long: their kernels start when the ones before have finished, as those of a step of many tokens
// do (common.cuh).  Those of fewer rows are chained if all blocks that quantise them are resident at once.  Us, chained and not: 65 rows
// x 4,096, 4,096 outputs 9.1 and 9.9, 256 rows 10.1 and 10.5, 84 x 14,336 21.9 and 23.2; beyond the rule 200 x 14,336 23.4 and 24.2,
// 400 x 4,096 12.7 and 13.0, 700 x 2,048, 2,048 outputs 9.9 both, 1,500 rows 11.4 and 10.7.
bool chained(long long rows, int K) { return rows <= 256 && rows * ((K + 255) / 256) <= 32LL * sm_count(); }

template <int NT, bool GROUPED>
int launch_nt(const Product& p, const void* rows, const void* W, cudaStream_t stream) {
    using L = Plan<NT>;
    static SharedLimit limit;
    if (const int e = limit.set(mx4_product_kernel<NT, GROUPED>, L::FIXED + 4 * (TABLE_EXPERTS + 1))) return e;
    CUtensorMap rows_map, w_map;
    if (!codes_map(rows, p.M, p.K, L::BOX, &rows_map) ||
        !codes_map(W, (long long)p.n_experts * p.N, p.K, UMMA_M, &w_map))
        return MLS_ERR_TENSOR_MAP;
    // (routed: the most units there can be, as every expert's last row tile may be partly filled)
    const long long tiles = GROUPED ? (long long)(p.M / NT) + (p.M < p.n_experts ? p.M : p.n_experts)
                                    : (long long)(p.M + NT - 1) / NT;
    const long long units = tiles * ((p.N + UMMA_M - 1) / UMMA_M);
    if (units > 0x7fffffffLL) return MLS_ERR_UNSUPPORTED;
    const int grid = (int)(units < sm_count() ? units : sm_count());
    const size_t smem = L::FIXED + (GROUPED ? 4 * (p.n_experts + 1) : 0);
    const int rc = chained(p.M, p.K)
                       ? launch_chained(mx4_product_kernel<NT, GROUPED>, dim3(grid), dim3(THREADS), smem, stream, p, rows_map, w_map)
                       : launch_plain(mx4_product_kernel<NT, GROUPED>, dim3(grid), dim3(THREADS), smem, stream, p, rows_map, w_map);
    return rc ? rc : launch_status();
}

template <int NT, bool GROUPED>
int launch_pair(const Product& p, const void* rows, const void* W, cudaStream_t stream) {
    using L = PairPlan<NT>;
    static_assert(L::FIXED + FEW_LEAST > 227 * 1024, "no block of a product of few rows beside a pair's");
    static SharedLimit limit;
    if (const int e = limit.set(mx4_pair_kernel<NT, GROUPED>, L::FIXED + 4 * (TABLE_EXPERTS + 1))) return e;
    const long long row_tiles = GROUPED ? p.M / TILE_ROWS + p.all_experts + 1 : (p.M + TILE_ROWS - 1) / TILE_ROWS;
    const long long w_tiles = (long long)p.n_experts * ((p.N + TILE_ROWS - 1) / TILE_ROWS);
    CUtensorMap rows_map, half_map, w_map, sf_rows_map, sf_w_map;
    if (!codes_map(rows, p.M, p.K, UMMA_M, &rows_map) || !codes_map(rows, p.M, p.K, UMMA_M / 2, &half_map) ||
        !codes_map(W, (long long)p.n_experts * p.N, p.K, NT / 2, &w_map) ||
        !scales_map(p.sf_a, row_tiles, p.K, 1, &sf_rows_map) || !scales_map(p.sf_w, w_tiles, p.K, 2, &sf_w_map))
        return MLS_ERR_TENSOR_MAP;
    const long long tiles = GROUPED ? (long long)(p.M / L::ROWS) + (p.M < p.n_experts ? p.M : p.n_experts)
                                    : (long long)(p.M + L::ROWS - 1) / L::ROWS;
    const long long units = tiles * ((p.N + NT - 1) / NT);
    if (units > 0x3fffffffLL) return MLS_ERR_UNSUPPORTED;
    const int most = sm_count() / 2, pairs = (int)(units < most ? units : most);
    const int rc = launch_plain(mx4_pair_kernel<NT, GROUPED>, dim3(2 * pairs), dim3(L::THREADS),
                                L::FIXED + (GROUPED ? 4 * (p.n_experts + 1) : 0), stream, p, rows_map, half_map, w_map, sf_rows_map, sf_w_map);
    return rc ? rc : launch_status();
}

// The ways of many rows, by the tile of a unit of work: 128 weights x 64 or 192 rows on one block, 256 rows x 192 or 256 weights on
// a pair (routed: 256 x 256 only).  Units are dealt out in rounds of one a block or pair; a round takes so long for every
// 256 of K, and so long for what its epilogue leaves visible (float32 sums of slots above all; pairs store them in whole lines).
// The cheapest way is taken: over 900 products of 17 to 2,048 rows or tokens and 256 to 14,336 of K, 0.5 % behind the fastest on
// average.  Measured, us, in the order 64 / 192 / 192 on pairs / 256 on pairs, rows quantised already:
//   256 rows x 14,336, 4,096 outputs       21.4 / 30.3 / 21.5 / 22.5     2,048 rows          125 / 82 / 54 / 42
//   128 x 4,096, 28,672 gated              23.4 / 16.0 / 20.1 / 17.1     2,048 rows          266 / 134 / 102 / 95
//   256 x 2,048, 2,048                     5.9 / 10.0 / 8.0 / 8.6        2,048 rows          15.6 / 15.7 / 11.6 / 9.3
// and routed, the whole call, 64 / 192 / pairs (8b: 64 experts of 4,096 x 1,408, 6 chosen; 1b: 32 of 2,048 x 1,024, 4 chosen):
//   8b, gate and up, 16 tokens  45 / 48 / 53, 600  94 / 84 / 90, 2,048  210 / 136 / 118
//   1b, down, 200 tokens        18.0 / 19.5 / 20.9, 600  29.3 / 35.0 / 26.7; 8b, 2,048 tokens  188 / 201 / 127
template <bool GROUPED>
int launch(const Product& p, const void* rows, const void* W, cudaStream_t stream) {
    const double k = (p.K + BK - 1) / BK, gated = p.unit == GATED ? 1 : 0, slots = GROUPED && p.unit == DOWN ? 1 : 0;
    // (routed: a prompt's experts have very unequal numbers of rows, most of the rows lie in experts of half as many again)
    const long long experts = p.M < p.n_experts ? p.M : p.n_experts;
    const long long each = GROUPED ? p.M * 3 / (2 * experts) + 1 : p.M;
    const long long sets = GROUPED ? experts : 1;
    auto rows_in = [&](int tile) { return (double)each / (double)((each + tile - 1) / tile); };
    auto cost = [&](long long row_tile, long long w_tile, int places, double per_k, double rest, double start) {
        const long long units = sets * ((each + row_tile - 1) / row_tile) * ((p.N + w_tile - 1) / w_tile);
        return start + (double)((units + places - 1) / places) * (k * per_k + rest);
    };
    const int blocks = sm_count(), pairs = blocks / 2;
    // (pairs store outputs at odd places row by row)
    const bool wide = p.width % (p.out_type == MLS_BF16 ? 16 : 8) == 0 && reinterpret_cast<uintptr_t>(p.out) % 32 == 0;
    const double odd = wide ? 0 : 0.8 + 0.5 * gated;
    const double t[4] = {cost(64, 128, blocks, 0.325, 0, 0),
                         cost(192, 128, blocks, 0.263 + 0.001 * rows_in(192), 0.9 + 7.7 * slots, 1.3),
                         GROUPED ? 1e30 : cost(256, 192, pairs, 0.289, 0.6 + 0.5 * gated + odd, 1.9),
                         GROUPED ? cost(256, 256, pairs, 0.342, 0.5 + 0.9 * gated, 0.1)
                                 : cost(256, 256, pairs, 0.24, 0.2 + 1.2 * gated + odd, 4.8)};
    int best = 0;
    for (int way = 1; way < 4; ++way)
        if (t[way] < t[best]) best = way;
    if (best == 0) return launch_nt<64, GROUPED>(p, rows, W, stream);
    if (best == 1) return launch_nt<192, GROUPED>(p, rows, W, stream);
    if constexpr (!GROUPED)
        if (best == 2) return launch_pair<192, false>(p, rows, W, stream);
    return launch_pair<256, GROUPED>(p, rows, W, stream);
}

// Chained, behind a quantisation too: one of a single round of blocks.  Longer ones let nobody start early (mx4.cu), so that no block that
// holds tensor memory and waits for its cluster becomes resident while they drain.
template <int NR, bool FUSED>
int launch_few(const FewProduct& p, const void* rows, const void* W, cudaStream_t stream) {
    using L = FewPlan<NR, FUSED>;
    static SharedLimit limit;
    if (const int e = limit.set(mx4_few_kernel<NR, FUSED>, L::total(FEW_SLICE))) return e;
    CUtensorMap rows_map, w_map;
    if (!codes_map(W, p.N, p.K, UMMA_M, &w_map)) return MLS_ERR_TENSOR_MAP;
    if (FUSED) rows_map = w_map;                                 // (not read)
    else if (!codes_map(rows, p.M, p.K, NR, &rows_map)) return MLS_ERR_TENSOR_MAP;
    const int kblocks = (p.K + BK - 1) / BK, slices = (kblocks + p.slice - 1) / p.slice;
    const int rc = launch_chained_cluster(mx4_few_kernel<NR, FUSED>, dim3(slices, (p.N + UMMA_M - 1) / UMMA_M),
                                          dim3(FEW_THREADS), L::total(p.slice), stream, dim3(slices, 1, 1), p, rows_map, w_map);
    return rc ? rc : launch_status();
}
}  // namespace

// One matrix.  rows_type >= 0: rows [M, K] of that type, ld values apart, that are quantised into a and sf_a first, or with
// `fused` within the product; rows_type < 0: a and sf_a are there.  slice > 0: the product of few rows (M <= 16 with `fused`, else
// 64), at most eight slices of so many times 256 of K.
static int product(int unit, const void* rows, int rows_type, long long ld, void* a, void* sf_a, const void* w, const void* sf_w,
                   void* out, int out_type, int M, int N, int K, int slice, int fused, int early, float alpha, float limit,
                   int* status, void* stream_) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0) return MLS_ERR_UNSUPPORTED;
    const cudaStream_t stream = (cudaStream_t)stream_;
    const int w_rows = unit == GATED ? pair_rows(N) : N;
    if (rows_type < 0 || slice <= 0) fused = 0;
    if (rows_type >= 0 && !fused) {
        const int rc = quantize_rows(rows, rows_type, ld, M, K, RowMap{M, 0, nullptr, nullptr, nullptr, 1, 0, 0}, (uint8_t*)a,
                                     (uint8_t*)sf_a, chained(M, K), stream);
        if (rc) return rc;
    }
    if (slice > 0) {
        const int kblocks = (K + BK - 1) / BK;
        if (M > (fused ? 16 : 64) || (fused && slice > FEW_SLICE) || (kblocks + slice - 1) / slice > FEW_SLICES ||
            (w_rows + UMMA_M - 1) / UMMA_M > 65535)
            return MLS_ERR_UNSUPPORTED;
        const int vec = reinterpret_cast<uintptr_t>(rows) % 16 == 0 && ld % (rows_type == MLS_BF16 ? 8 : 4) == 0;
        const FewProduct p{rows, out, (const uint8_t*)sf_w, (const uint8_t*)sf_a, ld, rows_type, vec, unit, out_type,
                           M, w_rows, K, N, slice, early, alpha, limit, status};
        if (fused) return launch_few<16, true>(p, a, w, stream);
        return M <= 16   ? launch_few<16, false>(p, a, w, stream)
               : M <= 32 ? launch_few<32, false>(p, a, w, stream)
                         : launch_few<64, false>(p, a, w, stream);
    }
    const Product p{out, (const uint8_t*)sf_w, (const uint8_t*)sf_a, nullptr, nullptr, nullptr, unit, 0, out_type,
                    1, 0, 1, M, w_rows, K, N, alpha, limit, status};
    return launch<false>(p, a, w, stream);
}

// Expert by expert: the slots of a routed step and w [E, 1 or 2, N, K].  The rows (sorted, or gathered from the tokens')
// are quantised into a and sf_a first, every slot's by itself, or with `places` (8 bytes a slot of scratch; gather only) every
// token's once for all of its slots.
static int expert_product(int unit, const void* rows, int rows_type, long long ld, int top, int gather, void* places, void* a,
                          void* sf_a, const void* w, const void* sf_w, void* out, int out_type,
                          int n_slots, int n_experts, int N, int K, const int* order, const int* idx, const int* offsets,
                          const float* weight, int scale, float alpha, float limit, int* status, void* stream_) {
    if (n_slots <= 0 || N <= 0 || n_experts <= 0) return 0;
    if (K <= 0 || top <= 0) return MLS_ERR_UNSUPPORTED;
    const cudaStream_t stream = (cudaStream_t)stream_;
    const RowMap map{n_slots, 0, order, idx, offsets, top, n_experts, gather};
    int rc;
    if (places) {
        rc = quantize_tokens(rows, rows_type, ld, n_slots / top, K, map, n_slots, places, (uint8_t*)a, (uint8_t*)sf_a, stream);
    } else {
        rc = quantize_rows(rows, rows_type, ld, n_slots, K, map, (uint8_t*)a, (uint8_t*)sf_a, chained(n_slots, K), stream);
    }
    if (rc) return rc;
    const int w_rows = unit == GATED ? pair_rows(N) : N;         // of an expert's weights
    // as many experts a launch as their table has room beside the stages
    for (int e0 = 0; e0 < n_experts; e0 += TABLE_EXPERTS) {
        const int n = n_experts - e0 < TABLE_EXPERTS ? n_experts - e0 : TABLE_EXPERTS;
        const size_t tiles = (size_t)e0 * ((w_rows + TILE_ROWS - 1) / TILE_ROWS);
        const Product p{out, (const uint8_t*)sf_w + tiles * atoms_of(K) * ATOM, (const uint8_t*)sf_a, order, offsets + e0,
                        weight, unit, scale, out_type, n, e0, n_experts, n_slots, w_rows, K, N, alpha, limit, status};
        rc = launch<true>(p, a, (const uint8_t*)w + (size_t)e0 * w_rows * pitch_of(K), stream);
        if (rc) return rc;
    }
    return 0;
}

MLS_API int mls_mx4_product(int unit, const void* rows, int rows_type, long long ld, void* a, void* sf_a, const void* w,
                            const void* sf_w, void* out, int out_type, int M, int N, int K, int slice, int fused, int early,
                            float alpha, float limit, int* status, void* stream) {
    return guarded([&] {
        return product(unit, rows, rows_type, ld, a, sf_a, w, sf_w, out, out_type, M, N, K, slice, fused, early, alpha, limit,
                       status, stream);
    });
}
MLS_API int mls_mx4_expert_product(int unit, const void* rows, int rows_type, long long ld, int top, int gather, void* places,
                                   void* a, void* sf_a, const void* w, const void* sf_w, void* out,
                                   int out_type, int n_slots, int n_experts, int N, int K, const int* order, const int* idx,
                                   const int* offsets, const float* weight, int scale, float alpha, float limit, int* status,
                                   void* stream) {
    return guarded([&] {
        return expert_product(unit, rows, rows_type, ld, top, gather, places, a, sf_a, w, sf_w, out, out_type, n_slots,
                              n_experts, N, K, order, idx, offsets, weight, scale, alpha, limit, status, stream);
    });
}
