// The down-projection of low-rank adapters on ConvRot INT8 activation codes,
// for gfx950.  No counterpart in the reference.
//
//   h[m][r] = scaling[a] * as[m] * sum_k code[m][k] * down[a][r][k],  a = the row's adapter
//
// The codes are those of the rotated activation x R, so `down` holds the rows
// of the adapter's matrix A rotated alike: (x R)(A R)^T = x A^T as R is
// orthonormal.  An int8 code is exact in bf16, so the product runs on
// v_mfma_f32_16x16x32_bf16 with fp32 sums; the up-projection follows in the
// INT8 GEMM's epilogue, where it joins the projection's fp32 value before the
// one rounding to bf16.
//
// A workgroup takes 16 to 64 rows and 16 to 64 ranks, its 8 waves a share of K
// each (they meet in LDS), and walks the distinct adapters of its rows; rows of
// one request lie together, so that is one adapter except at a border.  Each
// lane reads 16 codes of a row and the same 16 columns of a rank, which the
// MFMA takes as any order of K, so global reads are whole 64- and 128-byte
// pieces.  Few rows take the small tiles, and several workgroups (`slots`)
// share a tile's adapters; many rows of many adapters are sorted by it first.
//
// What bounds it: the loads of codes and ranks, half of the loop's time each;
// its waves wait for 43 to 79 % of their cycles.  32760 rows of 5120, rank 32:
// 51 us, 173 MB past the L2 (35 us of copy); 2050 rows, rank 64: 21 us, 54 MB.
// Whole 128-byte lines a load (lanes lc and lc + 8 exchanging halves) and the
// ranks of a row tile on one die were slower (134.5 -> 135.5, 132 -> 134.7 us
// with the GEMM at 2050 rows).
#include "adapters.h"

#include <algorithm>
#include <type_traits>

namespace tu {
namespace {


constexpr int kSortThreads = 1024;   // and the most adapters that are sorted
constexpr int64_t kLeastSorted = 256;  // rows
constexpr float kLargestBf16 = 0x1.fep127f;

// Tiles that the rows of `count` adapters fill at most.
int64_t sorted_tiles(int64_t m, int64_t count, int64_t rows) { return (m + rows - 1) / rows + std::min(count, m); }

__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t lo, uint32_t hi) {
    u32x4 out;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t w = j < 2 ? lo : hi;
        const int s = 16 * (j & 1);
        const float x = static_cast<float>(static_cast<int8_t>(w >> s));
        const float y = static_cast<float>(static_cast<int8_t>(w >> (s + 8)));
        out[j] = hw_bf16x2_bits(x, y);
    }
    return __builtin_bit_cast(bf16x8, out);
}

// The rows with an adapter, grouped by it: tiles of kRows places whose rows have
// one adapter, -1 in the places behind an adapter's last row.  One workgroup;
// which place of its adapter's tiles a row gets differs from run to run, and no
// result depends on it.
template <int kRows>
__global__ __launch_bounds__(kSortThreads) void adapter_sort_kernel(Adapters ad, int64_t m, int32_t *__restrict__ tiles,
                                                                    int32_t *__restrict__ places) {
    __shared__ int rows_of[kSortThreads], last[kSortThreads], first[kSortThreads];  // count <= kSortThreads
    const int t = threadIdx.x;
    rows_of[t] = 0;
    __syncthreads();
    for (int64_t row = t; row < m; row += kSortThreads) {
        const int a = adapter_of(ad.ids, ad.id_rows, ad.count, row, m);
        if (a >= 0) atomicAdd(&rows_of[a], 1);
    }
    __syncthreads();
    const int own = rows_of[t], need = (own + kRows - 1) / kRows;
    last[t] = need;
    __syncthreads();
    for (int d = 1; d < kSortThreads; d <<= 1) {
        const int add = t >= d ? last[t - d] : 0;
        __syncthreads();
        last[t] += add;
        __syncthreads();
    }
    first[t] = last[t] - need;
    for (int p = own; p < need * kRows; ++p) places[static_cast<int64_t>(first[t]) * kRows + p] = -1;
    if (t == kSortThreads - 1) *tiles = last[t];
    rows_of[t] = 0;
    __syncthreads();
    for (int64_t row = t; row < m; row += kSortThreads) {
        const int a = adapter_of(ad.ids, ad.id_rows, ad.count, row, m);
        if (a >= 0) places[static_cast<int64_t>(first[a]) * kRows + atomicAdd(&rows_of[a], 1)] = static_cast<int32_t>(row);
    }
}

// kRanks: ranks of a workgroup; kRowFrags: its 16-row fragments; kWaves: waves
// that share K; kSorted: the rows are those of a tile of adapter_sort_kernel.
template <int kRanks, int kRowFrags, int kWaves, bool kSorted>
__global__ __launch_bounds__(64 * kWaves) void adapter_down_kernel(const int8_t *__restrict__ a, const float *__restrict__ as,
                                                                const uint16_t *__restrict__ down,
                                                                const float *__restrict__ scaling, Adapters ad, int slots,
                                                                uint16_t *__restrict__ h, int64_t m, int64_t k,
                                                                const int32_t *__restrict__ tiles,
                                                                const int32_t *__restrict__ places) {
    constexpr int kFrags = kRanks / 16;
    constexpr int kRows = 16 * kRowFrags;
    __shared__ f32x4 sums[kWaves][kRowFrags * kFrags][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lc = lane & 15, g = lane >> 4;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
    const int r0 = static_cast<int>(blockIdx.y) * kRanks;
    const int slot = static_cast<int>(blockIdx.z);
    if (kSorted && static_cast<int>(blockIdx.x) >= *tiles) return;
    int64_t row_of[kRowFrags];  // this lane's row of a fragment
#pragma unroll
    for (int i = 0; i < kRowFrags; ++i) row_of[i] = kSorted ? places[row0 + 16 * i + lc] : row0 + 16 * i + lc;

    // the low lanes hold the tile's adapters (sorted: of the first row, which all have)
    const int64_t asked = kSorted ? max(places[row0 + lane % kRows], 0) : row0 + lane;
    const int id = lane < (kSorted ? 1 : kRows) ? adapter_of(ad.ids, ad.id_rows, ad.count, asked, m) : -1;
    uint64_t pending = __ballot(id >= 0);
    int ordinal = 0;
    while (pending) {
        const int which = __builtin_amdgcn_readlane(id, __builtin_ctzll(pending));
        const uint64_t mine = __ballot(id == which);
        pending &= ~mine;
        if (ordinal++ % slots != slot) continue;
        const uint16_t *dn = down + static_cast<int64_t>(which) * ad.rank * k;
        f32x4 acc[kFrags][kRowFrags];
#pragma unroll
        for (int f = 0; f < kFrags; ++f)
#pragma unroll
            for (int i = 0; i < kRowFrags; ++i) acc[f][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const int8_t *code[kRowFrags];
#pragma unroll
        for (int i = 0; i < kRowFrags; ++i) code[i] = a + max(min(row_of[i], m - 1), int64_t{0}) * k;
        const uint16_t *rank_row[kFrags];
#pragma unroll
        for (int f = 0; f < kFrags; ++f) rank_row[f] = dn + min(r0 + 16 * f + lc, ad.rank - 1) * k;
        // Steps of 64 columns; the last one takes zeros past K (a multiple of
        // 16).  The CU's other waves hide a step's loads better than two or
        // four steps of one wave in flight: 12.6, 13.3 and 13.7 us in all at 4
        // rows, 135.8, 137.6 and 141.5 at 2050, 850, 858 and 895 at 32760.
        auto step = [&](int64_t k0, auto tail) {
            int64_t kk = k0 + 16 * g;
            const bool in = !decltype(tail)::value || kk < k;
            kk = in ? kk : 0;
            u32x4 c[kRowFrags], d[kFrags][2];
#pragma unroll
            for (int i = 0; i < kRowFrags; ++i) c[i] = *reinterpret_cast<const u32x4 *>(code[i] + kk);
#pragma unroll
            for (int f = 0; f < kFrags; ++f)
#pragma unroll
                for (int e = 0; e < 2; ++e) d[f][e] = *reinterpret_cast<const u32x4 *>(rank_row[f] + kk + 8 * e);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                bf16x8 x[kRowFrags];
#pragma unroll
                for (int i = 0; i < kRowFrags; ++i) {
                    x[i] = codes_to_bf16(c[i][2 * e], c[i][2 * e + 1]);
                    if (!in) x[i] = __builtin_bit_cast(bf16x8, u32x4{0, 0, 0, 0});
                }
#pragma unroll
                for (int f = 0; f < kFrags; ++f) {
                    const u32x4 y = in ? d[f][e] : u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < kRowFrags; ++i)
                        acc[f][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, y), x[i], acc[f][i],
                                                                            0, 0, 0);
                }
            }
        };
        int64_t k0 = 64 * wave;
#pragma clang loop unroll(disable)
        for (; k0 + 64 <= k; k0 += 64 * kWaves) step(k0, std::false_type{});
        if (k0 < k) step(k0, std::true_type{});
#pragma unroll
        for (int f = 0; f < kFrags; ++f)
#pragma unroll
            for (int i = 0; i < kRowFrags; ++i) sums[wave][kRowFrags * f + i][lane] = acc[f][i];
        __syncthreads();
        // acc[f][i][r]: rank r0 + 16 f + 4 g + r of row row0 + 16 i + lc
        for (int t = wave; t < kRowFrags * kFrags; t += kWaves) {
            f32x4 v = sums[0][t][lane];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) v += sums[w][t][lane];
            const int f = t / kRowFrags, i = t % kRowFrags;
            int64_t row = row_of[0];
#pragma unroll
            for (int y = 1; y < kRowFrags; ++y) row = y == i ? row_of[y] : row;
            const int rank = r0 + 16 * f + 4 * g;
            // (the rank is a multiple of 8)
            if ((kSorted ? row >= 0 : (mine >> (16 * i + lc) & 1) != 0) && rank < ad.rank) {
                v *= scaling[which] * as[row];
                u32x2 hi, lo;
                // hi stops at bf16's largest number: what is past it, an infinity
                // too, is in lo (hi infinite would make lo infinity - infinity)
                auto held = [](float x) { return __builtin_amdgcn_fmed3f(x, -kLargestBf16, kLargestBf16); };
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    hi[e] = hw_bf16x2_bits(held(v[2 * e]), held(v[2 * e + 1]));
                    lo[e] = hw_bf16x2_bits(v[2 * e] - __uint_as_float(hi[e] << 16),
                                           v[2 * e + 1] - __uint_as_float(hi[e] & 0xffff0000u));
                }
                uint16_t *dst = h + h_at(row, ad.rank, rank);
                *reinterpret_cast<u32x2 *>(dst) = hi;
                *reinterpret_cast<u32x2 *>(dst + kLowTerm) = lo;
            }
        }
        __syncthreads();
    }
}

}  // namespace

int64_t adapters_workspace(int64_t m, int64_t rank) {
    // h, then the number of sorted tiles and their places
    const int64_t h = (m + 15) / 16 * ((rank + 31) / 32) * (2 * kLowTerm * 2);
    return h + (m >= kLeastSorted ? 16 + std::max(16 * sorted_tiles(m, kSortThreads, 16), 32 * sorted_tiles(m, kSortThreads, 32)) * 4 : 0);
}

int32_t launch_down(const int8_t *a, const float *a_scale, const uint16_t *down, const float *scaling,
                    const Adapters &ad, uint16_t *h, int32_t *sort, int64_t m, int64_t k, int cus, hipStream_t st) {
    // The largest tile that gives every CU a workgroup (four of the 32 rows for
    // one of 64: at 32760 rows of 5120, rank 32, 64 rows take 850 us with the
    // GEMM where 32 take 877), else the smallest.
    int rows = 32, ranks = ad.rank <= 16 ? 16 : ad.rank <= 32 ? 32 : 64;
    auto tiles = [&] { return (m + rows - 1) / rows * ((ad.rank + ranks - 1) / ranks); };
    while (tiles() < cus && ranks > 16) ranks /= 2;
    if (tiles() < cus) rows = 16;
    else if (ranks <= 32 && tiles() >= 4 * cus) rows = 64;
#define TU_DOWN(R, F, S) adapter_down_kernel<R, F, 8, S><<<grid, 512, 0, st>>>(a, a_scale, down, scaling, ad, slots, h, m, k, sort, sort + 4)
    // Requests of few rows: a tile walks every adapter among its rows, all of K
    // each time.  Where 16 rows have eight or more, or four and much work again,
    // the rows are sorted by their adapter first, by a launch of 5 to 11 us: with
    // it 1564 rows of 11760, 29 adapters of rank 40: 269 -> 27 us; 4000 of 5120,
    // 16 of rank 32: 148 -> 30; 300 of 2048, 32 of rank 64: 18.5 -> 10.7; 10027 of
    // 1344, 4 of rank 8 would go from 14 to 19 and is not sorted.  (Requests of 6
    // to 15 rows never are, though a tile of 64 rows may have 5 to 12 of them, nor
    // are more than 1024 adapters.)
    const int64_t walked = std::min<int64_t>(ad.count, (16 + ad.id_rows - 1) / ad.id_rows);
    if (ad.count <= kSortThreads && m >= kLeastSorted && m <= 0x7fffffff && walked >= 4 &&
        (walked >= 8 || (walked - 1) * m * k >= int64_t{1} << 26)) {
        rows = m / ad.count >= 32 ? 32 : 16;
        if (rows == 16) ranks = 16;
        const int slots = 1;
        const dim3 grid(static_cast<unsigned>(sorted_tiles(m, ad.count, rows)),
                        static_cast<unsigned>((ad.rank + ranks - 1) / ranks));
        if (rows == 16) adapter_sort_kernel<16><<<1, kSortThreads, 0, st>>>(ad, m, sort, sort + 4);
        else adapter_sort_kernel<32><<<1, kSortThreads, 0, st>>>(ad, m, sort, sort + 4);
        if (rows == 16) TU_DOWN(16, 1, true);
        else if (ranks == 16) TU_DOWN(16, 2, true);
        else if (ranks == 32) TU_DOWN(32, 2, true);
        else TU_DOWN(64, 2, true);
        return check_launch("tu_int8_gemm_adapters");
    }
    // two at least, so that a tile with a border between requests takes no longer
    const int slots = static_cast<int>(std::min<int64_t>(ad.count, std::min<int64_t>(16, std::max<int64_t>(2, cus / tiles()))));
    const dim3 grid(static_cast<unsigned>((m + rows - 1) / rows), static_cast<unsigned>((ad.rank + ranks - 1) / ranks),
                    static_cast<unsigned>(slots));
    if (rows == 16) TU_DOWN(16, 1, false);
    else if (rows == 64) {
        if (ranks == 16) TU_DOWN(16, 4, false);
        else TU_DOWN(32, 4, false);
    } else if (ranks == 16) TU_DOWN(16, 2, false);
    else if (ranks == 32) TU_DOWN(32, 2, false);
    else TU_DOWN(64, 2, false);
#undef TU_DOWN
    return check_launch("tu_int8_gemm_adapters");
}

}  // namespace tu
