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

namespace mls_mx4 {
constexpr int BLOCK = 32;
constexpr int TILE_ROWS = 128;
constexpr int ATOM = 512;

__host__ __device__ constexpr int pitch_of(int K) { return (K + BLOCK - 1) / BLOCK * (BLOCK / 2); }
__host__ __device__ constexpr int atoms_of(int K) { return 2 * ((K + 255) / 256); }
// Bytes from a tile's first atom to a row's four scales in its atom.
__host__ __device__ constexpr int row_in_atom(int r) { return (r & 31) * 16 + ((r >> 5) & 3) * 4; }

// Rows of the pairs [2, N, K] of gate and up matrices lie interleaved, 16 of the gate's and 16 of up's in turn (N filled up
// to a multiple of 16): an output's two sums are then 16 lanes of a warp apart.
__host__ __device__ constexpr int pair_rows(int N) { return (N + 15) / 16 * 32; }
__host__ __device__ constexpr int pair_row(int which, int n) { return n / 16 * 32 + which * 16 + n % 16; }

// Where row p of matrices of N rows each lies: its row of codes, the tile of its scales and its row in that.
struct Place {
    long long row, tile;
    int r;
};
__device__ __forceinline__ Place place_of(long long p, int N, bool pairs) {
    const long long mat = p / N;
    const int n = (int)(p - mat * N);
    const int rows = pairs ? pair_rows(N) : N, at = pairs ? pair_row((int)(mat & 1), n) : n;
    const long long m = pairs ? mat >> 1 : mat;
    return {m * rows + at, m * ((rows + TILE_ROWS - 1) / TILE_ROWS) + at / TILE_ROWS, at % TILE_ROWS};
}

// The sorted rows of a routed step: an expert's rows begin with a tile of their own.  Expert e's first tile is
// offsets[e] / 128 + e: with c rows behind offset o it takes ceil(c / 128) tiles, and (o + c) / 128 + 1 - o / 128,
// the distance to the next expert's, is never less.
__device__ __forceinline__ int first_tile(int offset, int e) { return offset / TILE_ROWS + e; }
}  // namespace mls_mx4
