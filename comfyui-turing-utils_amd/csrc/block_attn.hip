// Sage INT8 attention over listed key blocks (block-sparse attention) for
// gfx950.  No counterpart among the reference's kernels that this build
// restates; arithmetic and operand layouts are those of sage_attn.hip.
//
//   out_r = sum_j p_rj v_j / sum_j p_rj over the keys j of the listed blocks
//           that the row sees, p = 2^(s - m), m a running row maximum
//   s     = float(q8 . k8) * (sm_scale * log2 e) * q_scale * k_scale
// A list belongs to 128 query rows of one head and names blocks of 64 keys; an
// entry counts if it lies in [0, blocks) and is larger than every entry before
// it, so a block counts once whatever the list holds.  Rows at or past their
// sample's length, and rows that see no key, are zeros.
//
// MI355X mapping
//   * A unit of work is 128 query rows with their list, or a range of it: a
//     workgroup of 4 waves, 32 rows a wave, one wave per SIMD.  Two workgroups
//     share a CU (72 KiB of rings each at head_dim 128), and one's start-up and
//     end, 10 us beside 1.4 us a tile and so most of a short list, runs beside
//     the other's tiles.  (A persistent workgroup of two such groups with a
//     common barrier, in opposite phases by construction, took 1.40 us a tile
//     but stood still in both groups' start-ups: B1 H40 L32760 D128, 102 of 512
//     blocks, 3.13 ms, and 85 us against 65 for lists of 16.)
//   * The MFMA cluster has priority over the other workgroup's softmax, as in
//     the dense kernel: 3.00 ms at that shape, 3.07 without.
//   * K and V^T tiles stream through rings of three stages each.  A tile's K is
//     used one interval before its V^T, so in interval t (QK of tile t + 1, PV
//     of tile t) the loads of K(t + 3) and V^T(t + 2) go into the stages that
//     interval t - 1 read last, and have an interval to land.
//   * The list is compacted into LDS 256 entries at a time, by every wave for
//     itself (the same values), without a barrier.
//   * A grid that leaves workgroups' places empty splits its lists into
//     ranges, a unit each, merged by a second kernel.
#include <algorithm>

#include "attn_common.h"
#include "attn_plan.h"
#include "sage_tile.h"

namespace tu {
namespace {

constexpr int kBlockThreads = 256;
constexpr int kBlockRows = 128;
constexpr int kRing = 3;
constexpr int kSegment = 256;  // list entries compacted at a time
// Least factor of a masked tile's scores: 0 would make a masked one 0 * -inf.
// (2^(score * 1e-18) is 1 for every score.)
constexpr float kLeastFactor = 1e-18f;

struct BlockPlan {
    uint32_t nqb;    // query blocks of a head
    uint32_t blocks; // query blocks of all heads
    uint32_t width;  // entries of a list
    uint32_t parts;  // ranges of a list, a unit each
    uint32_t per;    // entries of a range
    uint32_t rows;   // partial rows of a query block
};

template <int D>
struct Ring {
    static constexpr int kV0 = kRing * Geo<D>::kKTileBytes;  // V^T stages follow the K stages
    static constexpr int kList = kRing * Geo<D>::kStageBytes;  // the compacted entries follow the rings
    static constexpr int kBytes = kList + kSegment * 4;
};

// Loads of one tile's K rows, or its V^T columns, into a ring stage (the two
// halves of issue_tile; same lanes, same swizzle).
#define TU_ISSUE_K_BODY(D)                                                                                          \
    constexpr int kK = Geo<D>::kKLoads;                                                                             \
    _Pragma("unroll") for (int i = 0; i < kK; ++i)                                                                  \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(krs, (lds_void *)(stage + (kK * wave + i) * 1024), 16,             \
                                                 gm.k_src[i] + key0 * k_sl, 0, 0, 0);
#define TU_ISSUE_V_BODY(D)                                                                                          \
    constexpr int kV = Geo<D>::kVLoads;                                                                             \
    _Pragma("unroll") for (int i = 0; i < kV; ++i)                                                                  \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(vrs, (lds_void *)(stage + (kV * wave + i) * 1024), 16, gm.v_src[i], \
                                                 key0 * 2, 0, 0);
#define TU_ISSUE(D)                                                                                                  \
    __device__ __forceinline__ void issue_k(int8_t *stage, __amdgpu_buffer_rsrc_t krs, const LaneGeom<D> &gm,         \
                                            uint32_t k_sl, uint32_t key0, int wave) {                                 \
        TU_ISSUE_K_BODY(D)                                                                                            \
    }                                                                                                                 \
    __device__ __forceinline__ void issue_v(int8_t *stage, __amdgpu_buffer_rsrc_t vrs, const LaneGeom<D> &gm,         \
                                            uint32_t key0, int wave) {                                                \
        TU_ISSUE_V_BODY(D)                                                                                            \
    }
TU_ISSUE(128)
TU_ISSUE(64)
// A tile's scale by a vector load whatever its address is: the waits of the
// main loop count it beside the tile's loads.
__device__ __forceinline__ float load_scale(__amdgpu_buffer_rsrc_t rs, int at) {
    return __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, at * 4, 0, 0));
}
#undef TU_ISSUE
#undef TU_ISSUE_K_BODY
#undef TU_ISSUE_V_BODY

// The largest value of 16 lanes, to all of them.
__device__ __forceinline__ float row_max16(float v) {
    // row_ror 8, 4, 2, 1
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xf, 0xf, true)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x124, 0xf, 0xf, true)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x122, 0xf, 0xf, true)));
    return fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x121, 0xf, 0xf, true)));
}

__device__ __forceinline__ int sample_end(const int32_t *lengths, uint32_t b, int64_t len) {
    return lengths ? min(max(lengths[b], 0), static_cast<int>(len)) : static_cast<int>(len);
}

// O^T += V^T P for a tile whose keys from `from` on may be behind the sample's
// end: their p is zero, but what stands there may be no number, so their values
// are zeroed as well.
template <int D>
__device__ __forceinline__ void pv_tail(const int8_t *stage, const LaneGeom<D> &gm, const bf16x8 (&p)[2][kQT],
                                        SoftmaxState<D> &st, const bf16x8 &ones, int from, int g) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        u32x4 keep;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int key = 32 * h + 8 * g + 2 * e;
            keep[e] = (key < from ? 0x0000ffffu : 0u) | (key + 1 < from ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int ds = 0; ds < Geo<D>::kDS; ++ds) {
            const u32x4 v = *reinterpret_cast<const u32x4 *>(stage + gm.v_rd[h] + ds * 16 * 128) & keep;
#pragma unroll
            for (int qt = 0; qt < kQT; ++qt)
                st.acc_o[ds][qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v), p[h][qt],
                                                                           st.acc_o[ds][qt], 0, 0, 0);
        }
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt)
            st.acc_l[qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[h][qt], st.acc_l[qt], 0, 0, 0);
    }
}

// kSplit: a range of a list writes the unnormalized O with each row's exponent
// base and row sum to `part` for block_merge_kernel.
// Workgroups of a CU: 2 fill the LDS at head_dim 128; at 64, 3 fill the
// registers (4 spill: 82 us for 53 at B2 H9 L6000 with 24 of 94 blocks).
template <int D>
constexpr int kWgsPerCu = D == 64 ? 3 : 2;

template <int D, bool kCausal, bool kSplit>
__global__ __launch_bounds__(kBlockThreads, kWgsPerCu<D>) void block_attn_kernel(
    const int8_t *__restrict__ q8, const float *__restrict__ q_scale, uint32_t blkq, uint32_t nbq,
    const int8_t *__restrict__ k8, const float *__restrict__ k_scale, int kscale_shift, uint32_t nbk,
    const uint16_t *__restrict__ vt, const int32_t *__restrict__ index, uint16_t *__restrict__ o, uint32_t hq,
    uint32_t groups, int64_t lq, int64_t lk, int64_t lpad, const int32_t *__restrict__ q_len,
    const int32_t *__restrict__ k_len, int64_t q_sb, int64_t q_sh, int64_t q_sl, int64_t k_sb, int64_t k_sh,
    int64_t k_sl, int64_t o_sb, int64_t o_sh, int64_t o_sl, float sm_log2, BlockPlan plan, float *__restrict__ part) {
    constexpr int kSl = Geo<D>::kKSlices;
    // a tile's loads, and the one of a later tile's scale beside them
    constexpr int kLoads = Geo<D>::kLoadsPerTile + 1;
    // One array: with several the compiler waits for all direct-to-LDS loads
    // before a tile's fragment reads.
    __shared__ __align__(1024) int8_t lds_mem[Ring<D>::kBytes];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4;
    const int lc = lane & 15;
    int8_t *lds = lds_mem;
    auto *list = reinterpret_cast<int *>(lds + Ring<D>::kList);
    // Each XCD owns a contiguous eighth of the units in the order K/V head,
    // sample, head, query block: neighbouring query blocks of a head, whose
    // lists are alike, and the heads of a K/V head share an L2, and a short
    // sample is spread over the XCDs (B2 H9 D64 of 6000 and 4000 tokens: 43 us;
    // sample by sample 54, as half of the XCDs have a third less to do).
    uint32_t id = xcd_chunk(blockIdx.x, gridDim.x), z = 0;
    if constexpr (kSplit) {
        z = id % plan.parts;
        id /= plan.parts;
    }
    const uint32_t qb = id % plan.nqb, order = id / plan.nqb, batch = plan.blocks / (plan.nqb * hq);
    const uint32_t b = order / groups % batch, hk = order / groups / batch;
    const uint32_t h = hk * groups + order % groups, bh = b * hq + h;
    id = bh * plan.nqb + qb;
    const int first = static_cast<int>(z * plan.per);
    const int end = min(static_cast<int>(plan.width), first + static_cast<int>(plan.per));
    const int32_t *entries = index + (static_cast<int64_t>(bh) * plan.nqb + qb) * plan.width;
    // Entries `at` .. of the list, 4 a lane (-1 past the unit's end).
    auto fetch = [&](int at, int (&e)[4]) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int i = at + 64 * c + lane;
            e[c] = entries[min(i, static_cast<int>(plan.width) - 1)];
            if (i >= end) e[c] = -1;
        }
    };
    int e[4];
    fetch(first, e);

    const uint32_t hkv = hq / groups;
    const int q_end = sample_end(q_len, b, lq), k_end = sample_end(k_len, b, lk);
    const int64_t qblock0 = static_cast<int64_t>(qb) * kBlockRows;
    const int64_t q0 = qblock0 + wave * kWaveQ;
    // blocks this query block can see at all, and the first that the sample's
    // end or a diagonal cuts
    int seen_end = k_end, masked_from = k_end / kBKey;
    if constexpr (kCausal) {
        seen_end = static_cast<int>(min<int64_t>(k_end, min<int64_t>(qblock0 + kBlockRows, q_end)));
        masked_from = static_cast<int>(min<int64_t>(masked_from, qblock0 / kBKey));
    }
    const int blocks = qblock0 < q_end ? (seen_end + kBKey - 1) / kBKey : 0;
    const int8_t *kp = k8 + b * k_sb + hk * k_sh;
    const uint16_t *vtp = vt + static_cast<int64_t>(b * hkv + hk) * D * lpad;
    const float *ks_row = k_scale + static_cast<int64_t>(b * hkv + hk) * nbk;
    const __amdgpu_buffer_rsrc_t srs = make_rsrc(ks_row, nbk * 4);
    // to the last row's end, whatever the stride (one row's may be anything)
    const __amdgpu_buffer_rsrc_t krs = make_rsrc(kp, static_cast<uint32_t>((lk - 1) * k_sl + D));
    const __amdgpu_buffer_rsrc_t vrs = make_rsrc(vtp, static_cast<uint32_t>(D * lpad * 2));
    const LaneGeom<D> gm = lane_geom<D>(wave, lane, k_sl, lpad);
    const uint32_t k_sl32 = static_cast<uint32_t>(k_sl);
    // K of a tile, or its V^T, into a ring stage
    auto load_k = [&](int stage, int block) {
        issue_k(lds + stage * Geo<D>::kKTileBytes, krs, gm, k_sl32, block * kBKey, wave);
    };
    auto load_v = [&](int stage, int block) {
        issue_v(lds + Ring<D>::kV0 + stage * Geo<D>::kVTileBytes, vrs, gm, block * kBKey, wave);
    };

    i32x4 qf[kQT][kSl];
    float qsc[kQT];
    {
        const int8_t *qp = q8 + b * q_sb + h * q_sh;
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) {
            const int64_t qi = min(q0 + 16 * qt + lc, lq - 1);
#pragma unroll
            for (int ds = 0; ds < kSl; ++ds)
                qf[qt][ds] = *reinterpret_cast<const i32x4 *>(qp + qi * q_sl + 64 * ds + 16 * g);
            // (a row behind the sample's end takes no part in what a wave's rows
            // decide together: when O is rescaled, how p is formed)
            qsc[qt] = qi < q_end ? q_scale[static_cast<int64_t>(bh) * nbq + static_cast<uint32_t>(qi) / blkq] : 0.0f;
        }
    }
    int before = -1;  // largest entry in front of the segment
    if constexpr (kSplit) {
        for (int i = lane; i < first; i += 64) before = max(before, entries[i]);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) before = max(before, __shfl_xor(before, d));
    }
    SoftmaxState<D> st;
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
        qsc[qt] *= sm_log2;
        st.m_used[qt] = kNoBase;
        st.acc_l[qt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ds = 0; ds < Geo<D>::kDS; ++ds) st.acc_o[ds][qt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const float largest_q = row_max16(fmaxf(qsc[0], qsc[1]));
    bf16x8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = static_cast<__bf16>(1.0f);
    i32x4 s[4][kQT];
    bf16x8 pb[2][kQT];

    for (int seg = first; seg < end; seg += kSegment) {
        if (seg > first) fetch(seg, e);
        // Compaction of the segment.  Ascending lists with nothing but -1 behind
        // them need no running maximum.
        bool ordered = true;
        int prev[4] = {};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (64 * c >= end - seg) break;  // all -1 from here on
            prev[c] = __shfl_up(e[c], 1);
            const int last = c ? __builtin_amdgcn_readlane(e[c - (c > 0)], 63) : before;
            if (lane == 0) prev[c] = last;
            ordered = ordered && (e[c] < 0 || (e[c] > prev[c] && (prev[c] >= 0 || (c == 0 && lane == 0))));
        }
        if (!__all(ordered)) {
            int top = before;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                int m = e[c];
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int other = __shfl_up(m, d);
                    if (lane >= d) m = max(m, other);
                }
                prev[c] = __shfl_up(m, 1);
                prev[c] = lane == 0 ? top : max(prev[c], top);
                top = max(top, __builtin_amdgcn_readlane(m, 63));
            }
        }
        int n = 0, whole = 0, top = before;
        float listed[4] = {};  // scales of the lane's entries, used when the first tile is done
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (64 * c >= end - seg) break;
            const bool counts = e[c] > prev[c] && e[c] >= 0 && e[c] < blocks;
            const uint64_t mask = __ballot(counts);
            if (counts) list[n + __builtin_popcountll(mask & ((1ull << lane) - 1))] = e[c];
            // (past the buffer's end: 0)
            listed[c] = load_scale(srs, counts ? e[c] >> kscale_shift : 0x1fffffff);
            n += __builtin_popcountll(mask);
            // tiles with masked keys stand last, as the list ascends
            whole += __builtin_popcountll(__ballot(counts && e[c] < masked_from));
            top = max(top, e[c]);
        }
        n = __builtin_amdgcn_readfirstlane(n);
        whole = __builtin_amdgcn_readfirstlane(whole);

        auto block_at = [&](int t) { return __builtin_amdgcn_readfirstlane(list[min(t, n - 1)]); };
        if (seg + kSegment < end) {
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) top = max(top, __shfl_xor(top, d));
            before = top;
        }
        if (n == 0) continue;

        auto softmax = [&](int t, float scale, auto mask_tag) {
            float f[kQT];
#pragma unroll
            for (int qt = 0; qt < kQT; ++qt) f[qt] = qsc[qt] * scale;
            if (decltype(mask_tag)::value && t >= whole) {
                const int key0 = block_at(t) * kBKey;
                const int key_lim = min(k_end - key0, kBKey);
                const int q_rel = static_cast<int>(max(min(q0 - key0, static_cast<int64_t>(kBKey)), static_cast<int64_t>(-kBlockRows)));
                mask_tile<kCausal>(s, key_lim, q_rel, g, lc);
                // a factor that is no number stays one, but not for a row that
                // sees nothing of the tile
#pragma unroll
                for (int qt = 0; qt < kQT; ++qt)
                    f[qt] = f[qt] < kLeastFactor || (kCausal && q_rel + 16 * qt + lc < 0) ? kLeastFactor : f[qt];
            }
            softmax_tile<decltype(mask_tag)::value>(s, f, st, pb);
        };
        auto uniform = [](float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); };
        // scale1 .. 3: scales of tiles t + 1 .. t + 3; block2, block3: blocks of
        // tiles t + 2 and t + 3
        const int block0 = block_at(0), block1 = block_at(1);
        int block2 = block_at(2), block3 = block_at(3);
        float scale0 = load_scale(srs, block0 >> kscale_shift), scale1 = load_scale(srs, block1 >> kscale_shift);
        float scale2 = load_scale(srs, block2 >> kscale_shift), scale3 = load_scale(srs, block3 >> kscale_shift);
        load_k(0, block0);
        load_v(0, block0);
        load_k(1, block1);
        load_v(1, block1);
        load_k(2, block2);
        // K(0), V(0), K(1) land, and with them every older load
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(Geo<D>::kLoadsPerTile));
        scale0 = uniform(scale0), scale1 = uniform(scale1), scale2 = uniform(scale2);
        wg_barrier();
        qk_tile(lds, gm, qf, s);
        softmax(0, scale0, std::true_type{});
        __builtin_amdgcn_s_waitcnt(lgkmcnt_imm(0));
        wg_barrier();  // K(0)'s stage is free for K(3)
        // Interval t: QK of tile t + 1 and PV of tile t, then the softmax of
        // tile t + 1.  At its end a wave waits for its loads of K(t + 2) and
        // V(t + 1), issued an interval ago.
        // A wave with a factor past kFarFactor leaves its tiles to the second
        // loop, which has the same barriers and fills the same stages: a test in
        // this loop costs 2 to 6 % at head_dim 64.
        const float largest_k = fmaxf(fmaxf(listed[0], listed[1]), fmaxf(listed[2], listed[3]));
        const int main_steps = __any(largest_q * largest_k > kFarFactor) ? 0 : max(0, min(n, whole) - 1);
        int s0 = 0, s1 = 1, s2 = 2;  // stages of tiles t, t + 1, t + 2
#pragma clang loop unroll(disable)
        for (int t = 0; t < main_steps; ++t) {
            mfma_cluster(lds + s1 * Geo<D>::kKTileBytes,
                         lds + Ring<D>::kV0 + s0 * Geo<D>::kVTileBytes - Geo<D>::kKTileBytes, gm, qf, s, pb, st, ones);
            const int e4 = list[min(t + 4, n - 1)];
            // K(t + 3) and V(t + 2) into stages last read in interval t - 1
            load_k(s0, block3);
            load_v(s2, block2);
            const float scale4 = load_scale(srs, e4 >> kscale_shift);
            softmax(t + 1, scale1, std::false_type{});
            block2 = block3, block3 = __builtin_amdgcn_readfirstlane(e4);
            const int free = s0;
            s0 = s1, s1 = s2, s2 = free;
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(kLoads));
            wg_barrier();
            scale1 = scale2, scale2 = uniform(scale3), scale3 = scale4;
        }
        // Masked tiles and the last one.
#pragma clang loop unroll(disable)
        for (int t = main_steps; t < n; ++t) {
            if (t + 3 < n) load_k(t % kRing, block_at(t + 3));
            if (t + 2 < n) load_v((t + 2) % kRing, block_at(t + 2));
            const int8_t *v = lds + Ring<D>::kV0 + (t % kRing) * Geo<D>::kVTileBytes - Geo<D>::kKTileBytes;
            if (t + 1 < n) qk_tile(lds + (t + 1) % kRing * Geo<D>::kKTileBytes, gm, qf, s);
            pv_tail(v, gm, pb, st, ones, k_end - block_at(t) * kBKey, g);
            if (t + 1 < n)
                softmax(t + 1, uniform(load_scale(srs, block_at(t + 1) >> kscale_shift)), std::true_type{});
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
            wg_barrier();
        }
    }

    // acc_o[ds][qt][r] = O[q0 + 16 qt + lc][16 ds + 4 g + r]; acc_l[qt][*] = l.
    if constexpr (kSplit) {
        // [parts][rows][D] fp32, then [parts][rows][2]
        const int64_t rows = static_cast<int64_t>(plan.blocks) * plan.rows;
        const int64_t row0 = z * rows + static_cast<int64_t>(id) * plan.rows + wave * kWaveQ;
        float *po = part + row0 * D;
        float *pml = part + plan.parts * rows * D + row0 * 2;
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) {
            const int r = 16 * qt + lc;
            if (q0 + r >= lq) continue;
#pragma unroll
            for (int ds = 0; ds < Geo<D>::kDS; ++ds)
                *reinterpret_cast<f32x4 *>(po + r * D + 16 * ds + 4 * g) = st.acc_o[ds][qt];
            // a row past its sample's end has seen nothing
            const bool in = q0 + r < q_end;
            if (g == 0) *reinterpret_cast<f32x2 *>(pml + r * 2) = f32x2{in ? st.m_used[qt] : kNoBase, in ? st.acc_l[qt][0] : 0.0f};
        }
        return;
    }
    uint16_t *op = o + b * o_sb + h * o_sh;
    const bool wide = ((reinterpret_cast<uintptr_t>(o) >> 1 | o_sb | o_sh | o_sl) & 7) == 0;
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
        const int64_t qi = q0 + 16 * qt + lc;
        const float l = st.acc_l[qt][0];
        // (a sum of 0 is a row that saw no key; one that is NaN stays NaN)
        const bool some = l != 0.0f && qi < q_end;
        const float inv = 1.0f / l;
#pragma unroll
        for (int ds = 0; ds < Geo<D>::kDS; ds += 2) {
            uint32_t w[2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const f32x4 a = st.acc_o[ds + i][qt];
                w[i][0] = some ? hw_bf16x2_bits(a[0] * inv, a[1] * inv) : 0;
                w[i][1] = some ? hw_bf16x2_bits(a[2] * inv, a[3] * inv) : 0;
            }
            // each lane ends with 8 contiguous channels of one row
            auto lo = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
            auto hi = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
            if (qi >= lq) continue;
            uint16_t *dst = op + qi * o_sl + 16 * (ds + (g & 1)) + 8 * (g >> 1);
            if (wide) {
                *reinterpret_cast<u32x4 *>(dst) = u32x4{lo[0], hi[0], lo[1], hi[1]};
            } else {
                reinterpret_cast<u32x2 *>(dst)[0] = u32x2{lo[0], hi[0]};
                reinterpret_cast<u32x2 *>(dst)[1] = u32x2{lo[1], hi[1]};
            }
        }
    }
}

// Merges the ranges of each row: M = max m_s, w_s = 2^(m_s - M),
// out = sum w_s O_s / sum w_s l_s, zeros where no range saw a key.  A range saw
// none where its l is 0 (its O may then be no number, and is left out); where
// its l is NaN the row is.
template <int D>
__global__ __launch_bounds__(256) void block_merge_kernel(const float *__restrict__ part, BlockPlan plan, uint32_t hq,
                                                          int64_t lq, uint16_t *__restrict__ o, int64_t o_sb,
                                                          int64_t o_sh, int64_t o_sl) {
    constexpr int kTpr = D / 8;  // threads per row, 8 channels each
    constexpr int kAhead = 8;    // ranges whose loads are in flight together
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / kTpr) + threadIdx.x / kTpr;
    const int d0 = (threadIdx.x % kTpr) * 8;
    const int64_t rows = static_cast<int64_t>(plan.blocks) * plan.rows;
    if (row >= rows) return;
    const uint32_t block = static_cast<uint32_t>(row / plan.rows);
    const uint32_t bh = block / plan.nqb;
    const int64_t q = static_cast<int64_t>(block % plan.nqb) * kBlockRows + row % plan.rows;
    if (q >= lq) return;
    const float *ml = part + plan.parts * rows * D;
    const int parts = static_cast<int>(plan.parts);
    float m = kNoBase, l = 0.0f, acc[8] = {};
    for (int p0 = 0; p0 < parts; p0 += kAhead) {
        f32x2 x[kAhead];
        f32x4 a[kAhead], c[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t at = min(p0 + u, parts - 1) * rows + row;
            x[u] = *reinterpret_cast<const f32x2 *>(ml + at * 2);
            a[u] = *reinterpret_cast<const f32x4 *>(part + at * D + d0);
            c[u] = *reinterpret_cast<const f32x4 *>(part + at * D + d0 + 4);
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) top = fmaxf(top, x[u][0]);
        const float old = __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= old;
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] *= old;
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (p0 + u >= parts || x[u][1] == 0.0f) continue;  // nothing seen in this range
            const float w = __builtin_amdgcn_exp2f(x[u][0] - m);
            l = __builtin_fmaf(w, x[u][1], l);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                acc[k] = __builtin_fmaf(w, a[u][k], acc[k]);
                acc[4 + k] = __builtin_fmaf(w, c[u][k], acc[4 + k]);
            }
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t *dst = o + (bh / hq) * o_sb + (bh % hq) * o_sh + q * o_sl + d0;
    u32x2 lo, hi;
    lo.x = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    lo.y = pack_bf16x2(acc[2] * inv, acc[3] * inv);
    hi.x = pack_bf16x2(acc[4] * inv, acc[5] * inv);
    hi.y = pack_bf16x2(acc[6] * inv, acc[7] * inv);
    reinterpret_cast<u32x2 *>(dst)[0] = lo;
    reinterpret_cast<u32x2 *>(dst)[1] = hi;
}

// Lists are split where the grid leaves places empty, into ranges of at least
// four entries: a round of units costs their tiles and a fixed part, and split
// the merge (in tiles of 1.4 us).  Splitting only the lists past a full round
// did not pay: a unit that has its CU to itself is faster (B1 H12 L8190 D128,
// 768 units: 97 us with the last 256 split, 87 without).
constexpr double kUnitTiles = 5.0;
constexpr double kMergeTiles = 4.0;

int64_t block_workspace(const BlockPlan &p, int64_t dim) {
    return p.parts > 1 ? static_cast<int64_t>(p.parts) * p.blocks * p.rows * (dim + 2) *
                             static_cast<int64_t>(sizeof(float))
                       : 0;
}

BlockPlan block_plan(int64_t batch, int64_t hq, int64_t lq, int64_t dim, int64_t width, int64_t cus, int64_t max_bytes) {
    BlockPlan p{};
    p.nqb = static_cast<uint32_t>((lq + kBlockRows - 1) / kBlockRows);
    p.blocks = static_cast<uint32_t>(batch * hq * p.nqb);
    p.rows = static_cast<uint32_t>(std::min<int64_t>(lq, kBlockRows));
    p.width = static_cast<uint32_t>(width);
    p.parts = 1;
    p.per = p.width;
    const int64_t slots = (dim == 64 ? kWgsPerCu<64> : kWgsPerCu<128>) * cus;
    double best = static_cast<double>(width) + kUnitTiles;
    for (int64_t parts = 2; p.blocks < slots && parts <= 64; ++parts) {
        const int64_t per = (width + parts - 1) / parts;
        if (per < 4) break;
        if ((width + per - 1) / per != parts) continue;
        BlockPlan c = p;
        c.parts = static_cast<uint32_t>(parts);
        c.per = static_cast<uint32_t>(per);
        if (block_workspace(c, dim) > max_bytes) break;
        const double cost = static_cast<double>((p.blocks * parts + slots - 1) / slots) * (per + kUnitTiles) + kMergeTiles;
        if (cost < best) {
            best = cost;
            p.parts = c.parts;
            p.per = c.per;
        }
    }
    return p;
}

}  // namespace
}  // namespace tu

extern "C" int64_t tu_sage_block_attn_workspace(int64_t batch, int64_t hq, int64_t lq, int64_t dim, int64_t width,
                                                int32_t cus) {
    using namespace tu;
    if (batch <= 0 || hq <= 0 || lq <= 0 || dim <= 0 || width <= 0 || cus <= 0) return 0;
    return block_workspace(block_plan(batch, hq, lq, dim, width, cus, INT64_MAX), dim);
}

extern "C" int32_t tu_sage_block_attn(const int8_t *q8, const float *q_scale, int64_t blkq, const int8_t *k8,
                                      const float *k_scale, int64_t blkk, const void *vt_bf16, int64_t lpad,
                                      const int32_t *index, int64_t width, void *o_bf16, int64_t batch, int64_t hq,
                                      int64_t hkv, int64_t lq, int64_t lk, int64_t dim, int64_t q_sb, int64_t q_sh,
                                      int64_t q_sl, int64_t k_sb, int64_t k_sh, int64_t k_sl, int64_t o_sb,
                                      int64_t o_sh, int64_t o_sl, const int32_t *q_lengths, const int32_t *k_lengths,
                                      float sm_scale, int32_t causal, int32_t cus, void *workspace,
                                      int64_t workspace_bytes, void *stream) {
    using namespace tu;
    TU_REQUIRE(dim == 64 || dim == 128, "block attention requires head_dim 64 or 128, got %lld",
               static_cast<long long>(dim));
    TU_REQUIRE(batch > 0 && hq > 0 && hkv > 0 && hq % hkv == 0, "block attention: hq must be a positive multiple of hkv");
    TU_REQUIRE(lq > 0 && lk > 0 && width > 0 && cus > 0 && lq <= 0x7fffff00 && lk <= 0x7fffff00 && width <= 0x3fffffff,
               "block attention sizes out of range");
    TU_REQUIRE(lpad >= lk && lpad % kBKey == 0, "block attention: V^T padded length must cover lk, multiple of 64");
    TU_REQUIRE(blkq > 0 && blkk > 0 && blkk % kBKey == 0 && ((blkk / kBKey) & (blkk / kBKey - 1)) == 0 &&
                   blkq <= 0x7fffffff && blkk <= 0x7fffffff,
               "block attention needs blkq > 0 and blkk = 64 * 2^n");
    TU_REQUIRE(k_sl >= 0 && q_sl >= 0 && lk * k_sl < (int64_t{1} << 32) && dim * lpad * 2 < (int64_t{1} << 32),
               "block attention: one head's K or V^T exceeds 4 GiB of addressable bytes");
    TU_REQUIRE(q8 && q_scale && k8 && k_scale && vt_bf16 && index && o_bf16, "block attention pointers must be non-null");
    TU_REQUIRE(sm_scale > 0.0f, "block attention sm_scale must be positive");
    TU_REQUIRE(q_sl % 16 == 0 && q_sh % 16 == 0 && q_sb % 16 == 0 && (reinterpret_cast<uintptr_t>(q8) & 15) == 0 &&
                   k_sl % 16 == 0 && k_sh % 16 == 0 && k_sb % 16 == 0 && (reinterpret_cast<uintptr_t>(k8) & 15) == 0,
               "block attention Q/K rows must be 16-byte aligned");
    TU_REQUIRE((reinterpret_cast<uintptr_t>(vt_bf16) & 15) == 0 && o_sl % 4 == 0 && o_sh % 4 == 0 && o_sb % 4 == 0 &&
                   (reinterpret_cast<uintptr_t>(o_bf16) & 7) == 0,
               "block attention V^T/O must be aligned");
    TU_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "block attention workspace must be 16-byte aligned");
    TU_REQUIRE(batch * hq <= 65535 && batch * hq * ((lq + kBlockRows - 1) / kBlockRows) <= 0x1fffffff,
               "block attention grid too large");
    const BlockPlan plan = block_plan(batch, hq, lq, dim, width, cus, workspace ? workspace_bytes : 0);
    const unsigned grid = plan.blocks * plan.parts;
    if (require_gfx950()) return -1;
    int kscale_shift = 0;
    while ((kBKey << kscale_shift) < blkk) ++kscale_shift;
    auto *part = static_cast<float *>(workspace);
    hipStream_t st = static_cast<hipStream_t>(stream);
#define TU_BLOCK_ATTN(D, CAUSAL, SPLIT)                                                                                \
    block_attn_kernel<D, CAUSAL, SPLIT><<<dim3(grid), kBlockThreads, 0, st>>>(                                              \
        q8, q_scale, static_cast<uint32_t>(blkq), static_cast<uint32_t>((lq + blkq - 1) / blkq), k8, k_scale,          \
        kscale_shift, static_cast<uint32_t>((lk + blkk - 1) / blkk), static_cast<const uint16_t *>(vt_bf16), index,    \
        static_cast<uint16_t *>(o_bf16), static_cast<uint32_t>(hq), static_cast<uint32_t>(hq / hkv), lq, lk, lpad,     \
        q_lengths, k_lengths, q_sb, q_sh, q_sl, k_sb, k_sh, k_sl, o_sb, o_sh, o_sl, sm_scale * kLog2e, plan, part)
#define TU_BLOCK_FORMS(D)                                                                                              \
    do {                                                                                                               \
        if (plan.parts > 1) {                                                                                          \
            if (causal) TU_BLOCK_ATTN(D, true, true);                                                                  \
            else TU_BLOCK_ATTN(D, false, true);                                                                        \
            constexpr int kRowsPerWg = 256 / (D / 8);                                                                  \
            const int64_t rows = static_cast<int64_t>(plan.blocks) * plan.rows;                                        \
            block_merge_kernel<D><<<dim3(static_cast<unsigned>((rows + kRowsPerWg - 1) / kRowsPerWg)), 256, 0, st>>>(  \
                part, plan, static_cast<uint32_t>(hq), lq, static_cast<uint16_t *>(o_bf16), o_sb, o_sh, o_sl);         \
        } else if (causal) {                                                                                           \
            TU_BLOCK_ATTN(D, true, false);                                                                             \
        } else {                                                                                                       \
            TU_BLOCK_ATTN(D, false, false);                                                                            \
        }                                                                                                              \
    } while (0)
    if (dim == 128) TU_BLOCK_FORMS(128);
    else TU_BLOCK_FORMS(64);
#undef TU_BLOCK_FORMS
#undef TU_BLOCK_ATTN
    return check_launch("tu_sage_block_attn");
}
