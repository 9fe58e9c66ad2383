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

template <int NR, bool FUSED>
__global__ void __launch_bounds__(FEW_THREADS)
mx4_few_kernel(const FewProduct p, const __grid_constant__ CUtensorMap rows_map, const __grid_constant__ CUtensorMap w_map) {
    few_block<NR, FUSED>(p, &rows_map, &w_map);
}

// Tensor maps by what they describe, as the other products keep theirs.
struct MapKey {
    const void* ptr;
    long long rows;
    int k, box_rows;
    bool operator<(const MapKey& o) const {
        return std::tie(ptr, rows, k, box_rows) < std::tie(o.ptr, o.rows, o.k, o.box_rows);
    }
};
bool codes_map(const void* ptr, long long rows, int K, int box_rows, CUtensorMap* out) {
    static std::map<MapKey, CUtensorMap> maps;
    static std::mutex lock;
    std::lock_guard<std::mutex> guard(lock);
    const MapKey key{ptr, rows, K, box_rows};
    auto it = maps.find(key);
    if (it == maps.end()) {
        if (maps.size() > 4096) maps.clear();
        EncodeTiledFn fn = encode_fn();
        if (!fn) return false;
        CUtensorMap m;
        const cuuint64_t size[2] = {(cuuint64_t)pitch_of(K), (cuuint64_t)rows}, stride[1] = {(cuuint64_t)pitch_of(K)};
        const cuuint32_t box[2] = {CODE_ROW, (cuuint32_t)box_rows}, step[2] = {1, 1};
        if (fn(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), size, stride, box, step,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
        it = maps.emplace(key, m).first;
    }
    *out = it->second;
    return true;
}

template <int NT, bool GROUPED>
int launch_nt(const Product& p, const void* rows, const void* W, cudaStream_t stream) {
    using L = Plan<NT>;
    static bool configured = false;
    if (!configured) {
        const cudaError_t e = cudaFuncSetAttribute(mx4_product_kernel<NT, GROUPED>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   L::FIXED + 4 * (TABLE_EXPERTS + 1));
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
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
    MLS_LAUNCH((mx4_product_kernel<NT, GROUPED>), dim3(grid), dim3(THREADS),
               L::FIXED + (GROUPED ? 4 * (p.n_experts + 1) : 0), stream, p, rows_map, w_map);
    return launch_status();
}

template <bool GROUPED>
int launch(const Product& p, const void* rows, const void* W, int average, cudaStream_t stream) {
    return average > 32 ? launch_nt<192, GROUPED>(p, rows, W, stream) : launch_nt<64, GROUPED>(p, rows, W, stream);
}

template <int NR, bool FUSED>
int launch_few(const FewProduct& p, const void* rows, const void* W, cudaStream_t stream) {
    using L = FewPlan<NR, FUSED>;
    static bool configured = false;
    if (!configured) {
        const cudaError_t e = cudaFuncSetAttribute(mx4_few_kernel<NR, FUSED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   L::total(FEW_SLICE));
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
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
MLS_API int mls_mx4_product(int unit, const void* rows, int rows_type, long long ld, void* a, void* sf_a, const void* w,
                            const void* sf_w, void* out, int out_type, int M, int N, int K, int slice, int fused, int early,
                            float alpha, float limit, int* status, void* stream_) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0) return MLS_ERR_UNSUPPORTED;
    const cudaStream_t stream = (cudaStream_t)stream_;
    const int w_rows = unit == GATED ? pair_rows(N) : N;
    if (rows_type < 0 || slice <= 0) fused = 0;
    if (rows_type >= 0 && !fused) {
        const int rc = quantize_rows(rows, rows_type, ld, M, K, RowMap{M, 0, nullptr, nullptr, nullptr, 1, 0, 0}, (uint8_t*)a,
                                     (uint8_t*)sf_a, stream);
        if (rc) return rc;
    }
    if (slice > 0) {
        const int kblocks = (K + BK - 1) / BK;
        if (M > (fused ? 16 : 64) || (fused && slice > FEW_SLICE) || (kblocks + slice - 1) / slice > 8 ||
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
                    1, 0, M, w_rows, K, N, alpha, limit, status};
    return launch<false>(p, a, w, M > 64 ? M : 0, stream);
}

// Expert by expert: the slots of a routed step and w [E, 1 or 2, N, K].  The rows (sorted, or gathered from the tokens')
// are quantised into a and sf_a first.
MLS_API int mls_mx4_expert_product(int unit, const void* rows, int rows_type, long long ld, int top, int gather, void* a,
                                   void* sf_a, const void* w, const void* sf_w, void* out, int out_type, int n_slots,
                                   int n_experts, int N, int K, const int* order, const int* idx, const int* offsets,
                                   const float* weight, int scale, float alpha, float limit, int* status, void* stream) {
    if (n_slots <= 0 || N <= 0 || n_experts <= 0) return 0;
    if (K <= 0 || top <= 0) return MLS_ERR_UNSUPPORTED;
    const int rc = quantize_rows(rows, rows_type, ld, n_slots, K, RowMap{n_slots, 0, order, idx, offsets, top, n_experts, gather},
                                 (uint8_t*)a, (uint8_t*)sf_a, (cudaStream_t)stream);
    if (rc) return rc;
    const int w_rows = unit == GATED ? pair_rows(N) : N;         // of an expert's weights
    // as many experts a launch as their table has room beside the stages
    for (int e0 = 0; e0 < n_experts; e0 += TABLE_EXPERTS) {
        const int n = n_experts - e0 < TABLE_EXPERTS ? n_experts - e0 : TABLE_EXPERTS;
        const size_t tiles = (size_t)e0 * ((w_rows + TILE_ROWS - 1) / TILE_ROWS);
        const Product p{out, (const uint8_t*)sf_w + tiles * atoms_of(K) * ATOM, (const uint8_t*)sf_a, order, offsets + e0,
                        weight, unit, scale, out_type, n, e0, n_slots, w_rows, K, N, alpha, limit, status};
        const int rc = launch<true>(p, a, (const uint8_t*)w + (size_t)e0 * w_rows * pitch_of(K), n_slots / n_experts,
                                    (cudaStream_t)stream);
        if (rc) return rc;
    }
    return 0;
}
