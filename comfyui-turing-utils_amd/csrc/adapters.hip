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
// A workgroup takes 32 rows and up to 64 ranks, its 8 waves a share of K each
// (they meet in LDS), and walks the distinct adapters of its rows; rows of one
// request lie together, so that is one adapter except at a border.  Each lane
// reads 16 codes of a row and the same 16 columns of a rank, which the MFMA
// takes as any order of K, so global reads are whole 64- and 128-byte pieces.
#include "adapters.h"

#include <algorithm>

namespace tu {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 32;

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

// kRanks: ranks of a workgroup (16, 32 or 64).
template <int kRanks>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(const int8_t *__restrict__ a, const float *__restrict__ as,
                                                                const uint16_t *__restrict__ down,
                                                                const float *__restrict__ scaling, Adapters ad,
                                                                DownPlan plan, float *__restrict__ h, int64_t m,
                                                                int64_t k) {
    constexpr int kFrags = kRanks / 16;
    __shared__ f32x4 sums[kWaves][2 * kFrags][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lc = lane & 15, g = lane >> 4;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
    const int r0 = static_cast<int>(blockIdx.y) * kRanks;
    const int part = static_cast<int>(blockIdx.z) / plan.slots, slot = static_cast<int>(blockIdx.z) % plan.slots;
    const int64_t k_begin = part * plan.per, k_end = min(k, k_begin + plan.per);

    // lanes 0 .. 31 hold the tile's adapters
    const int id = adapter_of(ad.ids, ad.id_rows, ad.count, row0 + (lane & 31), m);
    uint32_t pending = static_cast<uint32_t>(__ballot(id >= 0));
    int ordinal = 0;
    while (pending) {
        const int which = __builtin_amdgcn_readlane(id, __builtin_ctz(pending));
        const uint32_t mine = static_cast<uint32_t>(__ballot(id == which));
        pending &= ~mine;
        if (ordinal++ % plan.slots != slot) continue;
        const uint16_t *dn = down + static_cast<int64_t>(which) * ad.rank * k;
        f32x4 acc[kFrags][2];
#pragma unroll
        for (int f = 0; f < kFrags; ++f) acc[f][0] = acc[f][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const int8_t *code[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) code[i] = a + min(row0 + 16 * i + lc, m - 1) * k;
        const uint16_t *rank_row[kFrags];
#pragma unroll
        for (int f = 0; f < kFrags; ++f) rank_row[f] = dn + min(r0 + 16 * f + lc, ad.rank - 1) * k;
        for (int64_t k0 = k_begin + 64 * wave; k0 < k_end; k0 += 64 * kWaves) {
            const int64_t kk = k0 + 16 * g;
            const bool in = kk < k_end;  // K is a multiple of 16
            u32x4 c[2], d[kFrags][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) c[i] = in ? *reinterpret_cast<const u32x4 *>(code[i] + kk) : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int f = 0; f < kFrags; ++f)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    d[f][e] = in ? *reinterpret_cast<const u32x4 *>(rank_row[f] + kk + 8 * e) : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                bf16x8 x[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) x[i] = codes_to_bf16(c[i][2 * e], c[i][2 * e + 1]);
#pragma unroll
                for (int f = 0; f < kFrags; ++f)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        acc[f][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, d[f][e]), x[i],
                                                                            acc[f][i], 0, 0, 0);
            }
        }
#pragma unroll
        for (int f = 0; f < kFrags; ++f)
#pragma unroll
            for (int i = 0; i < 2; ++i) sums[wave][2 * f + i][lane] = acc[f][i];
        __syncthreads();
        // acc[f][i][r]: rank r0 + 16 f + 4 g + r of row row0 + 16 i + lc
        for (int t = wave; t < 2 * kFrags; t += kWaves) {
            f32x4 v = sums[0][t][lane];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) v += sums[w][t][lane];
            const int f = t >> 1, i = t & 1;
            const int64_t row = row0 + 16 * i + lc;
            const int rank = r0 + 16 * f + 4 * g;
            if ((mine >> (16 * i + lc) & 1) && rank < ad.rank) {  // the rank is a multiple of 8
                v *= scaling[which] * as[row];
                *reinterpret_cast<f32x4 *>(h + (part * m + row) * ad.rank + rank) = v;
            }
        }
        __syncthreads();
    }
}

}  // namespace

DownPlan down_plan(int64_t m, int64_t k, int64_t rank, int64_t count, int cus) {
    const int64_t tiles = (m + kRows - 1) / kRows * ((rank + 63) / 64);
    const int64_t slots = std::max<int64_t>(1, std::min({count, static_cast<int64_t>(cus) / tiles, int64_t{16}}));
    // a wave's share of a range is at least two steps of 64
    const int64_t parts = std::max<int64_t>(1, std::min({cus / (tiles * slots), k / (128 * kWaves), int64_t{8}}));
    const int64_t per = ((k + parts - 1) / parts + 63) / 64 * 64;
    return {static_cast<int>((k + per - 1) / per), static_cast<int>(slots), per};
}

int32_t launch_down(const int8_t *a, const float *a_scale, const uint16_t *down, const float *scaling,
                    const Adapters &ad, const DownPlan &plan, float *h, int64_t m, int64_t k, hipStream_t st) {
    const int ranks = ad.rank <= 16 ? 16 : ad.rank <= 32 ? 32 : 64;
    const dim3 grid(static_cast<unsigned>((m + kRows - 1) / kRows), static_cast<unsigned>((ad.rank + ranks - 1) / ranks),
                    static_cast<unsigned>(plan.parts * plan.slots));
#define TU_DOWN(R) adapter_down_kernel<R><<<grid, kThreads, 0, st>>>(a, a_scale, down, scaling, ad, plan, h, m, k)
    if (ranks == 16) TU_DOWN(16);
    else if (ranks == 32) TU_DOWN(32);
    else TU_DOWN(64);
#undef TU_DOWN
    return check_launch("tu_int8_gemm_adapters");
}

}  // namespace tu
