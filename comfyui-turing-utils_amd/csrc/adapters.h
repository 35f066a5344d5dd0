// What the two halves of a projection with low-rank adapters share: the
// down-projection (adapters.hip) writes its rows, the INT8 GEMM's epilogue
// (int8_gemm.hip) reads them.
#pragma once

#include "tu_common.h"

namespace tu {

// h holds a row's ranks as two bf16 terms (hi + lo is the fp32 sum to 2^-16 of
// it), scaled by the row's activation scale and its adapter's scaling, as the
// epilogue's MFMA reads them: [16 rows][32 ranks][term][row][32], a load of a
// wave being 1 KiB in one piece.  Rows without an adapter and ranks that pad the
// last 32 are not written.
struct Adapters {
    const uint16_t *h;
    const uint16_t *up;    // bf16 [count][n][up_rank]
    const int32_t *ids;    // adapter of rows i * id_rows .. (i + 1) * id_rows - 1
    int64_t id_rows;
    int rank, count;
    // The columns are parts of part_cols (a multiple of 16) side by side, and
    // those of part p see the up_rank ranks from p * up_rank on.
    int up_rank, part_cols;
};

// Place of a row's rank r in h; its low term lies kLowTerm values on.
constexpr int kLowTerm = 16 * 32;
__device__ __forceinline__ int64_t h_at(int64_t row, int rank, int r) {
    return ((row >> 4) * ((rank + 31) >> 5) + (r >> 5)) * (2 * kLowTerm) + (row & 15) * 32 + (r & 31);
}

// The adapter of a row, -1 for none (also where the id names no adapter).
__device__ __forceinline__ int adapter_of(const int32_t *ids, int64_t id_rows, int count, int64_t row, int64_t m) {
    if (row >= m) return -1;
    const int64_t i = (row | id_rows) >> 32 ? row / id_rows : static_cast<uint32_t>(row) / static_cast<uint32_t>(id_rows);
    const int a = ids[i];
    return static_cast<uint32_t>(a) < static_cast<uint32_t>(count) ? a : -1;
}

int32_t launch_down(const int8_t *a, const float *a_scale, const uint16_t *down, const float *scaling,
                    const Adapters &ad, uint16_t *h, int32_t *sort, int64_t m, int64_t k, int cus, hipStream_t st);

// Bytes of h and, behind it, of what launch_down sorts.
int64_t adapters_workspace(int64_t m, int64_t rank);

}  // namespace tu
