// One key tile of the INT8 Sage attention as a wave computes it: the tile's
// loads into LDS, S^T = K Q^T, masking, the softmax step and O^T += V^T P.
// Shared by the dense kernel (sage_attn.hip) and the one over selected key
// blocks (block_attn.hip); sage_attn.hip's head says how the parts fit together.
#pragma once

#include <type_traits>

#include "attn_common.h"

namespace tu {
namespace {

constexpr int kQT = 2;                   // 16-row query fragments per wave
constexpr int kWaveQ = 16 * kQT;         // query rows per wave
constexpr int kBKey = 64;                // keys per tile
constexpr float kRescaleSlack = 8.0f;        // log2 of the largest p allowed
constexpr float kFarFactor = 128.0f;         // f from which scores (22 bits times f) may pass 2^28
// Exponent base of a row that has seen no key yet, where a tile may have none
// for it: finite, so that such a tile gives 2^-inf = 0 and not a NaN, and below
// every finite score.
constexpr float kNoBase = -3.402823466e38f;

// Head-dim geometry (D = 64 or 128).  K tile: 64 keys x D bytes; V^T tile:
// D channels x 64 keys of bf16 (128-byte rows); group 0's 4 waves each move
// kKLoads + kVLoads 1 KiB blocks of a tile.
template <int D>
struct Geo {
    static_assert(D == 64 || D == 128, "head_dim 64 or 128");
    static constexpr int kKTileBytes = kBKey * D;
    static constexpr int kVTileBytes = D * kBKey * 2;
    static constexpr int kStageBytes = kKTileBytes + kVTileBytes;
    static constexpr int kKSlices = D / 64;  // 64-byte QK^T slices of a key row
    static constexpr int kDS = D / 16;       // 16-channel PV blocks
    static constexpr int kKLoads = kKTileBytes / 4096;
    static constexpr int kVLoads = kVTileBytes / 4096;
    static constexpr int kLoadsPerTile = kKLoads + kVLoads;
};

// K tile LDS row p holds key kperm(p): within each 32-key half, row
// 16 kt + i holds key 8 (i >> 2) + 4 kt + (i & 3).  The QK MFMA reads 16
// consecutive rows per 16-key block, so output row 4 g + r of block kt (of
// half h) is key 32 h + 8 g + 4 (kt & 1) + r, and each lane group g owns the
// 8 contiguous keys 32 h + 8 g .. +7: exactly one 16-byte V^T chunk.
__device__ __forceinline__ int kperm(int p) {
    const int i = p & 15, kt = (p >> 4) & 1;
    return (p & ~31) + 8 * (i >> 2) + 4 * kt + (i & 3);
}

// Per-lane constants of the tile loads and the MFMA operand reads.
template <int D>
struct LaneGeom {
    uint32_t k_src[Geo<D>::kKLoads];    // byte offset (from key0's row) of this lane's K source chunks
    uint32_t v_src[Geo<D>::kVLoads];    // byte offset (from key0's column) of this lane's V^T source chunks
    uint32_t k_rd[Geo<D>::kKSlices];    // LDS byte offset of the K operand of slice i
    uint32_t v_rd[2];                   // LDS byte offset of the V^T operand, half 0 / 1
};

// K rows of 128 B (D = 128) have their 16-byte chunks XOR-swizzled by row
// bits 1..3, rows of 64 B (D = 64) by row bits 2..3; either way the 16 lanes
// that read one chunk column of 16 consecutive rows hit distinct banks.
template <int D>
__device__ __forceinline__ LaneGeom<D> lane_geom(int wave, int lane, int64_t k_sl, int64_t lpad) {
    LaneGeom<D> gm;
    const int g = lane >> 4, lc = lane & 15, sw = (lc >> 1) & 7;
    if constexpr (D == 128) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = (2 * wave + i) * 8 + (lane >> 3);
            gm.k_src[i] = static_cast<uint32_t>(kperm(row) * k_sl + ((lane & 7) ^ ((row >> 1) & 7)) * 16);
            gm.k_rd[i] = static_cast<uint32_t>(lc * 128 + (((4 * i + g) ^ sw) << 4));
        }
    } else {
        const int row = wave * 16 + (lane >> 2);
        gm.k_src[0] = static_cast<uint32_t>(kperm(row) * k_sl + ((lane & 3) ^ ((row >> 2) & 3)) * 16);
        gm.k_rd[0] = static_cast<uint32_t>(lc * 64 + ((g ^ ((lc >> 2) & 3)) << 4));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        gm.v_rd[i] = static_cast<uint32_t>(Geo<D>::kKTileBytes + lc * 128 + (((4 * i + g) ^ sw) << 4));
#pragma unroll
    for (int i = 0; i < Geo<D>::kVLoads; ++i) {
        const int d = (Geo<D>::kVLoads * wave + i) * 8 + (lane >> 3);
        gm.v_src[i] = static_cast<uint32_t>((d * lpad + ((lane & 7) ^ ((d >> 1) & 7)) * 8) * 2);
    }
    return gm;
}

// Direct-to-LDS buffer loads of the K and V^T tiles at key0 into one ring
// stage.  Each buffer_load_dwordx4 ... lds moves 64 lanes x 16 B into 1 KiB of
// contiguous LDS; the K row permutation and the chunk swizzle come from the
// per-lane source offsets.  The tile's key offset goes into the per-lane
// offset, not the scalar one: the buffer range check covers only the
// per-lane offset, so K rows at or past lk (the range ends at lk rows) read
// as zeros instead of the bytes past the head's rows; those keys are masked
// by the softmax.  V^T is padded to whole tiles, so its key offset can stay
// scalar.
// One overload per head dim: the host compilation pass rejects a template of
// this function (the buffer builtins only exist for the device target), a
// plain device function it accepts.
#define TU_ISSUE_TILE_BODY(D)                                                                                      \
    constexpr int kK = Geo<D>::kKLoads, kV = Geo<D>::kVLoads;                                                      \
    _Pragma("unroll") for (int i = 0; i < kK; ++i)                                                                 \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(krs, (lds_void *)(stage + (kK * wave + i) * 1024), 16,            \
                                                 gm.k_src[i] + key0 * k_sl, 0, 0, 0);                              \
    _Pragma("unroll") for (int i = 0; i < kV; ++i)                                                                 \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(vrs, (lds_void *)(stage + Geo<D>::kKTileBytes + (kV * wave + i) * 1024), \
                                                 16, gm.v_src[i], key0 * 2, 0, 0);
__device__ __forceinline__ void issue_tile(int8_t *stage, __amdgpu_buffer_rsrc_t krs, __amdgpu_buffer_rsrc_t vrs,
                                           const LaneGeom<128> &gm, uint32_t k_sl, uint32_t key0, int wave) {
    TU_ISSUE_TILE_BODY(128)
}
__device__ __forceinline__ void issue_tile(int8_t *stage, __amdgpu_buffer_rsrc_t krs, __amdgpu_buffer_rsrc_t vrs,
                                           const LaneGeom<64> &gm, uint32_t k_sl, uint32_t key0, int wave) {
    TU_ISSUE_TILE_BODY(64)
}
#undef TU_ISSUE_TILE_BODY

// S^T for one tile: s[kt][qt][r] = biased score of key 32 (kt >> 1) + 8 g +
// 4 (kt & 1) + r and query 16 qt + lc of the wave.
template <int D>
__device__ __forceinline__ void qk_tile(const int8_t *stage, const LaneGeom<D> &gm,
                                        const i32x4 (&qf)[kQT][Geo<D>::kKSlices], i32x4 (&s)[4][kQT]) {
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
        i32x4 kf[Geo<D>::kKSlices];
#pragma unroll
        for (int i = 0; i < Geo<D>::kKSlices; ++i)
            kf[i] = *reinterpret_cast<const i32x4 *>(stage + gm.k_rd[i] + kt * 16 * D);
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) {
            i32x4 acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[0], qf[qt][0], i32x4{kBias, kBias, kBias, kBias},
                                                              0, 0, 0);
            if constexpr (D == 128) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[1], qf[qt][1], acc, 0, 0, 0);
            s[kt][qt] = acc;
        }
    }
}

// Softmax state of the wave: exponent base per query block, O^T and the row
// sums (l, accumulated by an MFMA against a ones operand so every lane ends
// with the complete sum for its query column).
template <int D>
struct SoftmaxState {
    float m_used[kQT];
    f32x4 acc_o[Geo<D>::kDS][kQT];
    f32x4 acc_l[kQT];
};

// Masks a tile's biased scores in place: masked keys (key >= key_lim, and for
// causal attention key > query) get the int bit pattern of -inf, which is
// below every biased score as an integer and stays -inf through the
// subtraction of the bias, so the row max ignores it and its p is 0.
template <bool kCausal>
__device__ __forceinline__ void mask_tile(i32x4 (&s)[4][kQT], int key_lim, int q_rel, int g, int lc) {
    constexpr int kNegInf = static_cast<int>(0xFF800000u);
    // key = c + 8 g with c a constant; key is masked iff c > t, with t the
    // lane's last visible key minus 8 g.  The select is done with integer
    // arithmetic (sign of t - c) to keep lane masks out of scalar registers.
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
        int t = key_lim - 1 - 8 * g;
        if constexpr (kCausal) t = min(t, q_rel + 16 * qt + lc - 8 * g);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int c = 32 * (kt >> 1) + 4 * (kt & 1) + r;
                const int m = (t - c) >> 31;  // all ones when masked
                s[kt][qt][r] = (s[kt][qt][r] & ~m) | (kNegInf & m);
            }
    }
}

// Softmax of one tile: lazy rescale of O and l, then P = 2^(dot f - m_used)
// rounded to bf16, packed as the PV B operands p[h][qt] (keys 32 h + 8 g ..
// + 7 of query 16 qt + lc).
//
// The exponent base m_used of a query row only moves when some score of the
// row exceeds it by more than kRescaleSlack; each lane tests its own 16
// scores (an integer max tree on the biased values), and only when some lane
// of the wave fails is the exact row maximum reduced across the 4 lanes that
// hold the row.
//
// x = dot f - m_used is formed as fma(biased, f, c) with
// c = -(1.5 * 2^23 f + m_used) when |c| < 2^12, which keeps the rounding of c
// below 2^-13 in the exponent; otherwise the bias is subtracted exactly first.
// kAnySize: where f is past kFarFactor the product is rounded before m_used, a
// rounded product too, is subtracted.  The FMA's exact product differs from
// m_used by up to half a step of it, and from scores of 2^31 on that leaves the
// exponent's range (all p infinite, or all 0).
template <bool kAnySize = false, int D>
__device__ __forceinline__ void softmax_tile(const i32x4 (&s)[4][kQT], const float (&f)[kQT], SoftmaxState<D> &st,
                                             bf16x8 (&p)[2][kQT]) {
    float mlane[kQT];
    bool need = false;
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
        int mi = imax3(s[0][qt][0], s[0][qt][1], s[0][qt][2]);
        mi = imax3(mi, s[0][qt][3], s[1][qt][0]);
        mi = imax3(mi, s[1][qt][1], s[1][qt][2]);
        mi = imax3(mi, s[1][qt][3], s[2][qt][0]);
        mi = imax3(mi, s[2][qt][1], s[2][qt][2]);
        mi = imax3(mi, s[2][qt][3], s[3][qt][0]);
        mi = imax3(mi, s[3][qt][1], s[3][qt][2]);
        mi = max(mi, s[3][qt][3]);
        mlane[qt] = (__int_as_float(mi) - kBiasF) * f[qt];
        need = need || (mlane[qt] > st.m_used[qt] + kRescaleSlack);
    }
    if (__any(need)) {
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) {
            const float m_new = fmaxf(st.m_used[qt], xmax_f32(mlane[qt]));
            // a row with no visible key yet keeps m_used = -inf and alpha = 1
            const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m_used[qt] - m_new);
            st.m_used[qt] = m_new;
            st.acc_l[qt] *= alpha;
#pragma unroll
            for (int ds = 0; ds < Geo<D>::kDS; ++ds) st.acc_o[ds][qt] *= alpha;
        }
    }
    float c[kQT];
    bool exact = false;
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
        c[qt] = -__builtin_fmaf(kBiasF, f[qt], st.m_used[qt]);
        exact = exact || !(fabsf(c[qt]) < 4096.0f);
    }
    // 0: an FMA on the biased score, 1: bias subtracted first, 2: product rounded as well
    auto make_p = [&](auto form_tag) {
        constexpr int kForm = decltype(form_tag)::value;
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) {
            const float nm = -st.m_used[qt];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 packed;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float p2[2];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int e = 2 * j + t;  // keys 32 h + 8 g + e
                        const float v = __int_as_float(s[2 * h + (e >> 2)][qt][e & 3]);
                        const float x = kForm == 0   ? __builtin_fmaf(v, f[qt], c[qt])
                                        : kForm == 1 ? __builtin_fmaf(v - kBiasF, f[qt], nm)
                                                     : (v - kBiasF) * f[qt] + nm;
                        p2[t] = __builtin_amdgcn_exp2f(x);
                    }
                    packed[j] =
                        __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{p2[0], p2[1]}), bf16x2_t));
                }
                p[h][qt] = __builtin_bit_cast(bf16x8, packed);
            }
        }
        // The exponentials run on a pipe of their own, an instruction every 16
        // cycles; left to itself the compiler puts eight of them in a row, and
        // the wave waits.  One between each two of the FMAs and conversions
        // instead: at head_dim 64, B1 H40 L32760 9.90 -> 9.07 ms, B1 H9 L6000
        // 95 -> 85 us.  At head_dim 128, where the other group's MFMAs are
        // twice as many, the runs are the better form (13.2 ms, 13.7 apart).
        if constexpr (D == 64) {
            constexpr int kFma = kForm + 1;
            __builtin_amdgcn_sched_group_barrier(0x002, 2 * kFma, 0);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, kFma, 0);
                __builtin_amdgcn_sched_group_barrier(0x400, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, kFma + 1, 0);
            }
        }
    };
    if (__any(exact)) {
        const bool far = kAnySize && __any(fmaxf(f[0], f[1]) > kFarFactor);
        if (__builtin_expect(far, 0)) make_p(std::integral_constant<int, 2>{});
        else make_p(std::integral_constant<int, 1>{});
    } else {
        make_p(std::integral_constant<int, 0>{});
    }
}

// O^T += V^T P and l += 1 P for one tile.
template <int D>
__device__ __forceinline__ void pv_tile(const int8_t *stage, const LaneGeom<D> &gm, const bf16x8 (&p)[2][kQT],
                                        SoftmaxState<D> &st, const bf16x8 &ones) {
    constexpr int kDS = Geo<D>::kDS;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        bf16x8 vf[kDS];
#pragma unroll
        for (int ds = 0; ds < kDS; ++ds)
            vf[ds] = *reinterpret_cast<const bf16x8 *>(stage + gm.v_rd[h] + ds * 16 * 128);
#pragma unroll
        for (int ds = 0; ds < kDS; ++ds)
#pragma unroll
            for (int qt = 0; qt < kQT; ++qt)
                st.acc_o[ds][qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[ds], p[h][qt], st.acc_o[ds][qt], 0, 0, 0);
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt)
            st.acc_l[qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[h][qt], st.acc_l[qt], 0, 0, 0);
    }
}

// MFMA cluster of a steady-state step: QK^T of the tile in kst and PV of the
// tile in vst, with the LDS fragment reads issued a group of MFMAs ahead of
// their first use.
template <int D>
__device__ __forceinline__ void mfma_cluster(const int8_t *kst, const int8_t *vst, const LaneGeom<D> &gm,
                                             const i32x4 (&qf)[kQT][Geo<D>::kKSlices], i32x4 (&s)[4][kQT],
                                             const bf16x8 (&p)[2][kQT], SoftmaxState<D> &st, const bf16x8 &ones) {
    constexpr int kDS = Geo<D>::kDS, kSl = Geo<D>::kKSlices;
    // This wave's MFMA cluster is the critical path of its interval: raise its
    // issue priority over the other group's softmax VALU on the same SIMD
    // (measured about 1 % faster; raising the softmax instead was slower).
    __builtin_amdgcn_s_setprio(3);
    i32x4 kf[4][kSl];
    bf16x8 va[kDS], vb[kDS];
    // first-slice K fragments first: the first QK^T MFMAs only need those
#pragma unroll
    for (int i = 0; i < kSl; ++i)
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) kf[kt][i] = *reinterpret_cast<const i32x4 *>(kst + gm.k_rd[i] + kt * 16 * D);
#pragma unroll
    for (int ds = 0; ds < kDS; ++ds) va[ds] = *reinterpret_cast<const bf16x8 *>(vst + gm.v_rd[0] + ds * 16 * 128);
    i32x4 z[4][kQT];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt)
            z[kt][qt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[kt][0], qf[qt][0], i32x4{kBias, kBias, kBias, kBias},
                                                              0, 0, 0);
    if constexpr (D == 128) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int qt = 0; qt < kQT; ++qt)
                s[kt][qt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[kt][kSl - 1], qf[qt][kSl - 1], z[kt][qt], 0, 0, 0);
    } else {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int qt = 0; qt < kQT; ++qt) s[kt][qt] = z[kt][qt];
    }
#pragma unroll
    for (int ds = 0; ds < kDS; ++ds) vb[ds] = *reinterpret_cast<const bf16x8 *>(vst + gm.v_rd[1] + ds * 16 * 128);
    // PV holds each V^T fragment (the A operand) for both query fragments,
    // as QK^T holds each K fragment: measured 1 % faster at B1 H40 L32760
    // than holding P across the V^T fragments (and QK^T holding Q across the
    // K fragments was 1 % slower).
#pragma unroll
    for (int ds = 0; ds < kDS; ++ds)
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt)
            st.acc_o[ds][qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[ds], p[0][qt], st.acc_o[ds][qt], 0, 0, 0);
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt)
        st.acc_l[qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[0][qt], st.acc_l[qt], 0, 0, 0);
#pragma unroll
    for (int ds = 0; ds < kDS; ++ds)
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt)
            st.acc_o[ds][qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb[ds], p[1][qt], st.acc_o[ds][qt], 0, 0, 0);
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt)
        st.acc_l[qt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[1][qt], st.acc_l[qt], 0, 0, 0);
    // Issue order, keeping at most 12 LDS reads in flight (the wait counter
    // holds 15; past that the compiler can only wait for all of them):
    // K reads, first QK^T MFMAs, first V^T half, second QK^T MFMAs (D = 128)
    // and 4 PV MFMAs, second V^T half, remaining PV MFMAs.
    if constexpr (D == 128) {
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 8, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 12, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 32, 0);
    } else {
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 9, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 15, 0);
    }
    __builtin_amdgcn_s_setprio(0);
}

}  // namespace
}  // namespace tu
