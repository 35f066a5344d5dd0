// Which key blocks a query block attends to: mean rows of the INT8 codes, the
// products of those means, and for each query block the `keep` key blocks with
// the largest product.  No counterpart in the reference's kernels that this
// build restates.
//
//   mq_i = mean over rows 128 i .. 128 i + 127 below the sample's length of
//          scale * code, mk_j = the same over keys 64 j .. 64 j + 63
//   S_ij = mq_i . mk_j
// The softmax scale is left out (it is positive), and so is any K smoothing
// mean (it adds the same to a whole row of S).
//
// A choice between two near scores is right or wrong, so what decides it is in
// 64 bits: code sums are integers, scale * sum is exact in fp64 (24 + 15 bits),
// and two orders of the fp64 sums differ by about 1e-15 of the score, where fp32
// would change about one choice in a hundred thousand.  But few scores are near
// the last one taken.  Each mean row is also kept as two bf16 terms, and three
// bf16 products give every score to within eps = 2^-13 |mq_i| max |mk_j|: those
// more than 2 eps above the approximate threshold are in, those more than 2 eps
// below are out, and only the others (one or two of 512) are computed in fp64.
//
// What bounds it at B1 H40 L32760 D128 (336 MB of codes): the means take 81 us,
// 384 MB read and written at 4.7 TB/s, and the choice 39 us: 16 of products, 6
// for the scores' way back from LDS, 9 of search, 8 of fp64 scores and lists;
// past the products it is bound by instructions, comparisons and bit counts.
// With every score from fp64 MFMAs and a search bit by bit it was 69 + 73 us.
#include "tu_common.h"
#include "attn_plan.h"

namespace tu {
namespace {

typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int kQBlock = 128;  // rows of a query block
constexpr int kKBlock = 64;   // keys of a key block
constexpr int kThreads = 256;
constexpr int kSelectThreads = 512;
constexpr int kTileQ = 16;         // query blocks of a scoring workgroup (one MFMA's rows)
constexpr int kMaxLdsBlocks = 2048;  // key blocks whose keys fit LDS (16 rows of 8 KiB)

// The approximate scores' error over |mq_i| |mk_j|: with x = hi + lo + r, |lo|
// <= 2^-8 |x| and |r| <= 2^-16 |x|, the products left out are under 3 * 2^-16 of
// |q| |k|, and 384 sums in fp32, rounded or cut, under 2^-14.4 of it: 2^-13.4.
constexpr float kScoreError = 0x1p-13f;

constexpr int kFewOpen = 8;  // undecided blocks that 16 lanes score each

// What block_mean_kernel leaves of one side's blocks: fp64 mean rows, the same
// as bf16 terms hi and lo, and their lengths (rounded up).  The terms stand as
// the MFMA reads them, [head][16 blocks][term, 32 channels][block][32]: a load
// of a wave is 1 KiB in one piece, where rows of 16 blocks gave 64-byte pieces
// (B1 H40, 256 x 512 blocks: 56 -> 46 us).
struct Means {
    double *mean;
    uint16_t *split;
    float *norm;
};

// Of a block's channel 0 in `split`; 32 channels on lie 512 values on, lo 16 D.
template <int D>
__device__ __forceinline__ int64_t split_at(uint32_t bh, uint32_t blk, uint32_t blocks) {
    return (static_cast<int64_t>(bh) * ((blocks + 15) / 16) + blk / 16) * 32 * D + blk % 16 * 32;
}

// One side's codes and what its blocks need.
struct Side {
    const int8_t *codes;
    const float *scale;
    const int32_t *lengths;  // per batch entry, or null
    int64_t s_b, s_h, s_l;
    uint32_t heads, len, group, scales;  // group: tokens per scale
    uint32_t blocks;
};

__device__ __forceinline__ int sample_end(const int32_t *lengths, uint32_t b, int len) {
    return lengths ? min(max(lengths[b], 0), len) : len;
}

// Mean row of one block, a wave's work: each load brings 64 x 16 codes, whole
// rows of 16 codes per lane, and the codes are added as unsigned bytes (biased
// by 128) in packed 16-bit halves, 6 instructions per 4 codes; at the end of a
// scale's rows the integer sums go to fp64 times the scale.
template <int D, int kRows>
__device__ __forceinline__ void block_mean(const Side &s, uint32_t bh, uint32_t blk, const Means &out, int lane) {
    constexpr int kLanesPerRow = D / 16;
    constexpr int kRpl = 64 / kLanesPerRow;  // rows per load
    constexpr int kLoads = kRows / kRpl;
    const uint32_t b = bh / s.heads, h = bh % s.heads;
    const int t0 = static_cast<int>(blk * kRows);
    const int valid = max(0, min(sample_end(s.lengths, b, static_cast<int>(s.len)) - t0, kRows));
    const int64_t at = static_cast<int64_t>(bh) * s.blocks + blk;
    const int8_t *base = s.codes + b * s.s_b + h * s.s_h + (lane % kLanesPerRow) * 16;
    const float *scale = s.scale + static_cast<int64_t>(bh) * s.scales;
    const int r0 = lane / kLanesPerRow;
    u32x4 raw[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        // rows at or past the sample's end read a valid row and count as zero
        const int64_t row = min(t0 + i * kRpl + r0, static_cast<int>(s.len) - 1);
        raw[i] = *reinterpret_cast<const u32x4 *>(base + row * s.s_l);
        if (i * kRpl + r0 >= valid) raw[i] = u32x4{0, 0, 0, 0};
    }
    // Loads that share one scale: all rows of a load do where the scale's
    // groups begin at loads, else every load is multiplied by its lane's scale.
    const uint32_t g = s.group;
    const int per = kRows % g == 0 && g % kRpl == 0 ? static_cast<int>(g) / kRpl : g % kRows == 0 ? kLoads : 1;
    double acc[16] = {};
    uint32_t even[4] = {0, 0, 0, 0}, odd[4] = {0, 0, 0, 0};
    int since = 0;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t x = raw[i][w] ^ 0x80808080u;
            even[w] += x & 0x00ff00ffu;
            odd[w] += (x >> 8) & 0x00ff00ffu;
        }
        ++since;
        if (since == per || i == kLoads - 1) {
            const int row = min(t0 + i * kRpl + r0, static_cast<int>(s.len) - 1);
            // a scale behind the sample's end may be no number
            const bool some = (i + 1 - since) * kRpl + r0 < valid;
            const double f = some ? static_cast<double>(scale[static_cast<uint32_t>(row) / g]) : 0.0;
            const int bias = 128 * since;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int c[4] = {static_cast<int>(even[w] & 0xffffu) - bias, static_cast<int>(odd[w] & 0xffffu) - bias,
                                  static_cast<int>(even[w] >> 16) - bias, static_cast<int>(odd[w] >> 16) - bias};
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[4 * w + e] = __builtin_fma(f, static_cast<double>(c[e]), acc[4 * w + e]);
                even[w] = odd[w] = 0;
            }
            since = 0;
        }
    }
    // Across the lanes that hold the same channels: each step hands half of a
    // lane's channels to its partner.
    int n = 16, first = 0;
#pragma unroll
    for (int m = kLanesPerRow; m < 64; m <<= 1) {
        n /= 2;
        const bool up = (lane & m) != 0;
        first += up ? n : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j >= n) break;
            const double send = up ? acc[j] : acc[j + n];
            const double keep = up ? acc[j + n] : acc[j];
            acc[j] = keep + __shfl_xor(send, m);
        }
    }
    const double count = static_cast<double>(max(valid, 1));
    const int c0 = (lane % kLanesPerRow) * 16 + first;
    uint16_t *split = out.split + split_at<D>(bh, blk, s.blocks) + (c0 >> 5) * 512 + (c0 & 31);
    float square = 0.0f;
    if constexpr (D == 128) {  // two channels a lane
        const f64x2 m = {acc[0] / count, acc[1] / count};
        *reinterpret_cast<f64x2 *>(out.mean + at * D + c0) = m;
        const uint32_t hi = hw_bf16x2_bits(static_cast<float>(m[0]), static_cast<float>(m[1]));
        const uint32_t lo = hw_bf16x2_bits(static_cast<float>(m[0] - static_cast<double>(bf16_bits_to_f32(hi & 0xffffu))),
                                           static_cast<float>(m[1] - static_cast<double>(bf16_bits_to_f32(hi >> 16))));
        *reinterpret_cast<uint32_t *>(split) = hi;
        *reinterpret_cast<uint32_t *>(split + 16 * D) = lo;
        square = static_cast<float>(m[0] * m[0] + m[1] * m[1]);
    } else {
        const double m = acc[0] / count;
        out.mean[at * D + c0] = m;
        const uint32_t hi = hw_bf16x2_bits(static_cast<float>(m), 0.0f) & 0xffffu;
        const uint32_t lo = hw_bf16x2_bits(static_cast<float>(m - static_cast<double>(bf16_bits_to_f32(hi))), 0.0f);
        split[0] = static_cast<uint16_t>(hi);
        split[16 * D] = static_cast<uint16_t>(lo & 0xffffu);
        square = static_cast<float>(m * m);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) square += __shfl_xor(square, d);
    if (lane == 0) out.norm[at] = __builtin_sqrtf(square) * 1.00001f;
}

// One wave per block: the query blocks first, then the key blocks.
template <int D>
__global__ __launch_bounds__(kThreads) void block_mean_kernel(Side q, Side k, uint32_t q_tasks, uint32_t tasks, Means mq,
                                                              Means mk) {
    const uint32_t task = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (task >= tasks) return;
    if (task < q_tasks) {
        block_mean<D, kQBlock>(q, task / q.blocks, task % q.blocks, mq, lane);
    } else {
        const uint32_t t = task - q_tasks;
        block_mean<D, kKBlock>(k, t / k.blocks, t % k.blocks, mk, lane);
    }
}

// A score as an integer of the same order: NaN below every number, -0 as 0.
__device__ __forceinline__ uint64_t order_key(double v) {
    if (v != v) return 1;
    const uint64_t x = __builtin_bit_cast(uint64_t, v + 0.0);
    return x ^ ((x >> 63) ? ~0ull : 1ull << 63);
}

struct Choice {
    uint32_t keep, sink, local, width;
    int causal;
};

// Key blocks that a query block sees: a prefix, as lengths and the causal
// mask both cut the end off.
__device__ __forceinline__ int visible_blocks(int qb, int q_end, int k_end, int causal) {
    if (qb * kQBlock >= q_end) return 0;
    const int end = causal ? min(k_end, min((qb + 1) * kQBlock, q_end)) : k_end;
    return (end + kKBlock - 1) / kKBlock;
}

__device__ __forceinline__ bool forced(int qb, int j, const Choice &c) {
    const int w = static_cast<int>(c.local);
    return j < static_cast<int>(c.sink) || (w > 0 && j >= 2 * qb - (w - 1) && j <= 2 * qb + w);
}

// Visits a lane's keys 0 .. kParts - 1, held in registers, or `parts` of them
// (kParts 0).
template <int kParts, typename Visit>
__device__ __forceinline__ void each_part(int parts, Visit visit) {
    if constexpr (kParts > 0) {
#pragma unroll
        for (int p = 0; p < kParts; ++p) visit(p);
    } else {
        for (int p = 0; p < parts; ++p) visit(p);
    }
}

// A threshold that `take` keys reach (key(p) is the lane's key of block 64 p +
// lane), or more where keys equal it: found bit by bit, counting the keys at or
// above it, until the count fits.  More than `take` keys are above zero.
template <int kParts, typename Int, typename Key>
__device__ __forceinline__ Int threshold(int take, int parts, Key key) {
    Int t = 0;
    for (int bit = 8 * sizeof(Int) - 1; bit >= 0; --bit) {
        const Int cand = t | static_cast<Int>(1) << bit;
        int count = 0;
        each_part<kParts>(parts, [&](int p) { count += __builtin_popcountll(__ballot(key(p) >= cand)); });
        if (count >= take) t = cand;
        if (count == take) break;
    }
    return t;
}

// Writes the blocks whose keys are above t and, lower ones first, as many of
// those equal to it as make `take`, in ascending order with -1 behind.
template <int kParts, typename Int, typename Key>
__device__ __forceinline__ void write_row(Int t, int take, int width, int lane, int parts, Key key,
                                          int32_t *__restrict__ out) {
    int above = 0;
    each_part<kParts>(parts, [&](int p) { above += __builtin_popcountll(__ballot(key(p) > t)); });
    const int allowed = take - above;
    const uint64_t below = (1ull << lane) - 1;
    int ties = 0, pos = 0;
    each_part<kParts>(parts, [&](int p) {
        const Int v = key(p);
        const uint64_t equal = __ballot(v == t);
        const bool chosen = v > t || (v == t && ties + __builtin_popcountll(equal & below) < allowed);
        const uint64_t mask = __ballot(chosen);
        if (chosen) out[pos + __builtin_popcountll(mask & below)] = 64 * p + lane;
        ties += __builtin_popcountll(equal);
        pos += __builtin_popcountll(mask);
    });
    for (int i = pos + lane; i < width; i += 64) out[i] = -1;
}

// S of one query block and the lane's key block in fp64.
template <int D>
__device__ __forceinline__ double exact_score(const double *__restrict__ mq, const double *__restrict__ mk) {
    double s = 0.0;
#pragma unroll 8
    for (int d = 0; d < D; d += 2) {
        const f64x2 x = *reinterpret_cast<const f64x2 *>(mq + d), y = *reinterpret_cast<const f64x2 *>(mk + d);
        s = __builtin_fma(x[0], y[0], s);
        s = __builtin_fma(x[1], y[1], s);
    }
    return s;
}

// The same by 16 lanes, every one a part of the channels.
template <int D>
__device__ __forceinline__ double group_score(const double *__restrict__ mq, const double *__restrict__ mk, int lc) {
    double s = 0.0;
#pragma unroll
    for (int d = 2 * lc; d < D; d += 32) {
        const f64x2 x = *reinterpret_cast<const f64x2 *>(mq + d), y = *reinterpret_cast<const f64x2 *>(mk + d);
        s = __builtin_fma(x[0], y[0], s);
        s = __builtin_fma(x[1], y[1], s);
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) s += __shfl_xor(s, d);
    return s;
}

template <int kBlocks>
constexpr int kChooseThreads = kBlocks <= 128 ? 1024 : 512;

// Approximate scores of 16 query blocks and all key blocks of one head into
// LDS; then a wave per query block makes the choice.
// Up to 512 key blocks three workgroups fit a CU, so that the 640 of 40 heads
// and 256 query blocks all run at once (two: 65 us for 60).
template <int D, int kBlocks>
__global__ __launch_bounds__(kChooseThreads<kBlocks>, kBlocks <= 512 ? 6 : 2) void block_choose_kernel(
    Means mq, Means mk, Choice c, uint32_t hq, uint32_t groups, uint32_t nqb, uint32_t nkb, int lq, int lk,
    const int32_t *__restrict__ q_len, const int32_t *__restrict__ k_len, int32_t *__restrict__ index) {
    constexpr int kWaves = kChooseThreads<kBlocks> / 64, kParts = kBlocks / 64, kChunks = D / 32;
    __shared__ float scores[kTileQ * kBlocks];  // [query block][key block]
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lc = lane & 15, g = lane >> 4;
    const uint32_t tiles = (nqb + kTileQ - 1) / kTileQ;
    // A head's tiles, and the heads of a K/V head, on one die, whose L2 reads the
    // key blocks once; a short sample's tiles are spread over all dies.
    const uint32_t tile = xcd_chunk(blockIdx.x, gridDim.x), order = tile / tiles, hkv = hq / groups;
    const uint32_t batch = gridDim.x / (tiles * hq), b = order / groups % batch;
    const uint32_t h = order / groups / batch * groups + order % groups, bh = b * hq + h;
    const int i0 = static_cast<int>(tile % tiles) * kTileQ;
    const int q_end = sample_end(q_len, b, lq), k_end = sample_end(k_len, b, lk);
    const int64_t q_row = static_cast<int64_t>(bh) * nqb, k_row = static_cast<int64_t>(b * hkv + h / groups) * nkb;
    // (rows behind the last block hold anything and are not used)
    const uint16_t *qs = mq.split + split_at<D>(bh, i0, nqb) + lc * 32 + 8 * g;
    const uint16_t *k_split = mk.split + split_at<D>(b * hkv + h / groups, 0, nkb) + lc * 32 + 8 * g;
    bf16x8 a[2][kChunks];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < kChunks; ++u) a[t][u] = *reinterpret_cast<const bf16x8 *>(qs + t * 16 * D + 512 * u);
    // no row of the tile sees more than its last one
    const int last = min(i0 + kTileQ, static_cast<int>(nqb)) - 1;
    const int most = c.causal ? (min(k_end, (last + 1) * kQBlock) + kKBlock - 1) / kKBlock : (k_end + kKBlock - 1) / kKBlock;
    float longest = 0.0f;
#pragma unroll
    for (int p = 0; p < kParts; ++p)
        longest = fmaxf(longest, 64 * p + lane < most ? mk.norm[k_row + 64 * p + lane] : 0.0f);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) longest = fmaxf(longest, __shfl_xor(longest, d));
    constexpr int kRowsOfWave = kTileQ / kWaves;
    float norms[kRowsOfWave];
#pragma unroll
    for (int x = 0; x < kRowsOfWave; ++x) norms[x] = mq.norm[q_row + min(i0 + wave + x * kWaves, static_cast<int>(nqb) - 1)];
    for (int j0 = 16 * wave; j0 < most; j0 += 16 * kWaves) {
        const int j = j0 + lc;
        const uint16_t *ks = k_split + static_cast<int64_t>(j0) * 2 * D;
        bf16x8 x[2][kChunks];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < kChunks; ++u) x[t][u] = *reinterpret_cast<const bf16x8 *>(ks + t * 16 * D + 512 * u);
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < kChunks; ++u) {
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0][u], x[1][u], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1][u], x[0][u], acc, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < kChunks; ++u) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0][u], x[0][u], acc, 0, 0, 0);
        // acc[r]: query block i0 + 4 g + r and key block j
#pragma unroll
        for (int r = 0; r < 4; ++r) scores[(4 * g + r) * kBlocks + j] = acc[r];
    }
    __syncthreads();
    for (int x = 0; x < kRowsOfWave; ++x) {
        const int r = wave + x * kWaves, i = i0 + r;
        if (i >= static_cast<int>(nqb)) break;
        const int n = visible_blocks(i, q_end, k_end, c.causal);
        const int take = min(static_cast<int>(c.keep), n), width = static_cast<int>(c.width);
        int32_t *out = index + (q_row + i) * c.width;
        if (take == n) {
            for (int p = lane; p < width; p += 64) out[p] = p < n ? p : -1;
            continue;
        }
        // a block out of sight is below every score, a forced one above
        float v[kParts], lo = INFINITY, hi = -INFINITY;
        bool finite = true;
        int force = 0;
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
            const int j = 64 * p + lane;
            const float y = j < n ? scores[r * kBlocks + j] : 0.0f;
            const bool first = j < n && forced(i, j, c);
            finite = finite && __builtin_fabsf(y) < INFINITY;
            v[p] = j >= n ? -INFINITY : first ? INFINITY : y;
            lo = j < n && !first ? fminf(lo, y) : lo;
            hi = j < n && !first ? fmaxf(hi, y) : hi;
            force += __builtin_popcountll(__ballot(first));
        }
        if (force >= take) {
            write_row<kParts>(1u, take, width, lane, 0, [&](int p) { return v[p] == INFINITY ? 1u : 0u; }, out);
            continue;
        }
        const float norm = x == 0 ? norms[0] : norms[kRowsOfWave - 1];
        float eps = kScoreError * norm * longest;
        const double *row = mq.mean + (q_row + i) * D;
        // Sums in fp32 that left its range, or neared its smallest numbers, or
        // means of NaN say nothing: all blocks that are not forced are open.
        if (!(__all(finite) && norm > 0x1p-40f && norm < 0x1p60f && longest > 0x1p-40f && longest < 0x1p60f)) {
            each_part<kParts>(0, [&](int p) {
                const int j = 64 * p + lane;
                if (j < n && !forced(i, j, c)) v[p] = 0.0f;
            });
            lo = hi = eps = 0.0f;
        }
        // The last score taken lies in lo .. hi: by interpolation and halving
        // in turn, until the two are eps apart or just `take` reach lo.
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            lo = fminf(lo, __shfl_xor(lo, d));
            hi = fmaxf(hi, __shfl_xor(hi, d));
        }
        int at_lo = n, at_hi = force;  // keys that reach them
        for (bool halve = false; hi - lo > eps; halve = !halve) {
            const float part = halve ? 0.5f
                                     : __builtin_amdgcn_fmed3f((static_cast<float>(at_lo - take) + 0.5f) *
                                                                   __builtin_amdgcn_rcpf(static_cast<float>(at_lo - at_hi)),
                                                               0.0625f, 0.9375f);
            const float mid = lo + (hi - lo) * part;
            int count = 0;
            each_part<kParts>(0, [&](int p) { count += __builtin_popcountll(__ballot(v[p] >= mid)); });
            if (count >= take) lo = mid, at_lo = count;
            else hi = mid, at_hi = count;
            if (count == take) {
                hi = INFINITY;
                each_part<kParts>(0, [&](int p) { hi = v[p] >= mid ? fminf(hi, v[p]) : hi; });
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) hi = fminf(hi, __shfl_xor(hi, d));
                lo = hi;
            }
        }
        // blocks above `in` are taken, those below `outside` not
        const float in = hi + 2.25f * eps, outside = lo - 2.25f * eps;
        int sure = 0, open = 0;
        each_part<kParts>(0, [&](int p) {
            sure += __builtin_popcountll(__ballot(v[p] > in));
            open += __builtin_popcountll(__ballot(v[p] <= in && v[p] >= outside));
        });
        if (sure + open == take) {
            write_row<kParts>(1u, take, width, lane, 0, [&](int p) { return v[p] >= outside ? 1u : 0u; }, out);
            continue;
        }
        // A few open blocks: scored four at a time, 16 lanes each; lane t then
        // holds the t-th and counts those before it.
        if (open <= kFewOpen) {
            int mine[kFewOpen / 4] = {}, found = 0;  // lane / 16's blocks
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
                uint64_t left = __ballot(v[p] <= in && v[p] >= outside);
                for (; left != 0; left &= left - 1, ++found)
                    if ((lane >> 4) == (found & 3)) mine[found >> 2] = 64 * p + __builtin_ctzll(left);
            }
            double s[kFewOpen / 4];
#pragma unroll
            for (int q = 0; q < kFewOpen / 4; ++q)
                s[q] = __shfl(group_score<D>(row, mk.mean + (k_row + mine[q]) * D, lc), 16 * (lane & 3));
            const uint64_t own = order_key(lane < 4 ? s[0] : s[1]);
            int before = 0;
            for (int t = 0; t < open; ++t) {
                const uint64_t other = __shfl(own, t);
                before += other > own || (other == own && t < lane) ? 1 : 0;
            }
            const uint64_t win = __ballot(lane < open && before < take - sure);
            found = 0;
            each_part<kParts>(0, [&](int p) {
                const bool undecided = v[p] <= in && v[p] >= outside;
                const uint64_t all = __ballot(undecided);
                const int place = found + __builtin_popcountll(all & ((1ull << lane) - 1));
                if (undecided) v[p] = win >> place & 1 ? INFINITY : -INFINITY;
                found += __builtin_popcountll(all);
            });
            write_row<kParts>(1u, take, width, lane, 0, [&](int p) { return v[p] > in ? 2u : 0u; }, out);
            continue;
        }
        // Many: one to a lane.  (One way for a row: equal scores stay equal.)
        uint64_t key[kParts];
        each_part<kParts>(0, [&](int p) { key[p] = v[p] > in ? ~0ull : v[p] >= outside ? 1ull : 0ull; });
#pragma clang loop unroll(disable)
        for (int p = 0; p < kParts; ++p) {
            bool undecided = false;
#pragma unroll
            for (int y = 0; y < kParts; ++y) undecided = y == p ? key[y] == 1ull : undecided;
            if (!__any(undecided)) continue;
            const uint64_t e = undecided ? order_key(exact_score<D>(row, mk.mean + (k_row + 64 * p + lane) * D)) : 0ull;
#pragma unroll
            for (int y = 0; y < kParts; ++y) key[y] = y == p && undecided ? e : key[y];
        }
        const uint64_t t = threshold<kParts, uint64_t>(take, 0, [&](int p) { return key[p]; });
        write_row<kParts>(t, take, width, lane, 0, [&](int p) { return key[p]; }, out);
    }
}

// For more key blocks than LDS holds: every score of 16 query blocks and all
// key blocks of one head in fp64, as ordered keys in `scores`.  Lane group g
// reads channels 8 u + 2 g and the next for the products 2 u and 2 u + 1, 64
// bytes of a row per load.
template <int D>
__global__ __launch_bounds__(kSelectThreads) void block_score_kernel(const double *__restrict__ mean_q,
                                                                     const double *__restrict__ mean_k, Choice c,
                                                                     uint32_t hq, uint32_t groups, uint32_t nqb,
                                                                     uint32_t nkb, int lq, int lk,
                                                                     const int32_t *__restrict__ q_len,
                                                                     const int32_t *__restrict__ k_len,
                                                                     uint64_t *__restrict__ scores) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lc = lane & 15, g = lane >> 4;
    const uint32_t tiles = (nqb + kTileQ - 1) / kTileQ;
    const uint32_t bh = blockIdx.x / tiles;
    const int i0 = static_cast<int>(blockIdx.x % tiles) * kTileQ;
    const uint32_t b = bh / hq, h = bh % hq, hkv = hq / groups;
    const int q_end = sample_end(q_len, b, lq), k_end = sample_end(k_len, b, lk);
    const double *mq = mean_q + (static_cast<int64_t>(bh) * nqb + min(i0 + lc, static_cast<int>(nqb) - 1)) * D + 2 * g;
    const double *mk = mean_k + static_cast<int64_t>(b * hkv + h / groups) * nkb * D + 2 * g;
    f64x2 a[D / 8];
#pragma unroll
    for (int u = 0; u < D / 8; ++u) a[u] = *reinterpret_cast<const f64x2 *>(mq + 8 * u);
    // no row of the tile sees more than its last one
    const int last = min(i0 + kTileQ, static_cast<int>(nqb)) - 1;
    const int most = c.causal ? (min(k_end, (last + 1) * kQBlock) + kKBlock - 1) / kKBlock : (k_end + kKBlock - 1) / kKBlock;
    for (int j0 = 16 * wave; j0 < most; j0 += 16 * (kSelectThreads / 64)) {
        const int j = j0 + lc;
        const double *kr = mk + static_cast<int64_t>(min(j, static_cast<int>(nkb) - 1)) * D;
        f64x4 acc = {0.0, 0.0, 0.0, 0.0};
        f64x2 x[D / 8];
#pragma unroll
        for (int u = 0; u < D / 8; ++u) x[u] = *reinterpret_cast<const f64x2 *>(kr + 8 * u);
#pragma unroll
        for (int u = 0; u < D / 8; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(a[u][e], x[u][e], acc, 0, 0, 0);
        // acc[r] = S of query block i0 + 4 r + g and key block j
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + 4 * r + g;
            if (i < static_cast<int>(nqb) && j < static_cast<int>(nkb))
                scores[(static_cast<int64_t>(bh) * nqb + i) * nkb + j] =
                    j >= visible_blocks(i, q_end, k_end, c.causal) ? 0ull : forced(i, j, c) ? ~0ull : order_key(acc[r]);
        }
    }
}

// The choice from keys in memory, a wave per query block.
__global__ __launch_bounds__(kThreads) void choose_kernel(const uint64_t *__restrict__ scores, Choice c, uint32_t hq,
                                                          uint32_t nqb, uint32_t nkb, uint32_t rows, int lq, int lk,
                                                          const int32_t *__restrict__ q_len,
                                                          const int32_t *__restrict__ k_len,
                                                          int32_t *__restrict__ index) {
    const uint32_t id = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (id >= rows) return;
    const uint32_t b = id / nqb / hq;
    const int n = visible_blocks(static_cast<int>(id % nqb), sample_end(q_len, b, lq), sample_end(k_len, b, lk), c.causal);
    const uint64_t *row = scores + static_cast<int64_t>(id) * nkb;
    auto key = [&](int p) { return 64 * p + lane < n ? row[64 * p + lane] : 0ull; };
    const int take = min(static_cast<int>(c.keep), n), parts = (n + 63) / 64;
    const uint64_t t = take < n ? threshold<0, uint64_t>(take, parts, key) : 1ull;
    write_row<0>(t, take, static_cast<int>(c.width), lane, parts, key, index + static_cast<int64_t>(id) * c.width);
}

int64_t blocks_of(int64_t len, int64_t block) { return (len + block - 1) / block; }

// Values of bf16 terms of every head, the heads padded to 16 blocks.
int64_t split_values(int64_t heads, int64_t blocks, int64_t dim) { return heads * ((blocks + 15) / 16) * 32 * dim; }

// fp64 mean rows, their bf16 terms and their lengths (padded to 16 bytes), then the ordered keys where they do not fit LDS.
int64_t select_workspace(int64_t batch, int64_t hq, int64_t hkv, int64_t lq, int64_t lk, int64_t dim) {
    const int64_t nqb = blocks_of(lq, kQBlock), nkb = blocks_of(lk, kKBlock);
    const int64_t rows = batch * (hq * nqb + hkv * nkb);
    const int64_t split = split_values(batch * hq, nqb, dim) + split_values(batch * hkv, nkb, dim);
    return rows * dim * 8 + split * 2 + (rows * 4 + 15) / 16 * 16 + (nkb > kMaxLdsBlocks ? batch * hq * nqb * nkb * 8 : 0);
}

template <int D>
int32_t launch_select(const Side &q, const Side &k, int64_t batch, int64_t hq, int64_t hkv, const Choice &c, void *ws,
                      int32_t *index, hipStream_t st) {
    const uint32_t nqb = q.blocks, nkb = k.blocks;
    const int64_t q_tasks = batch * hq * nqb, tasks = q_tasks + batch * hkv * nkb;
    auto *mean = static_cast<double *>(ws);
    auto *split = reinterpret_cast<uint16_t *>(mean + tasks * D);
    auto *k_split = split + split_values(batch * hq, nqb, D);
    auto *norm = reinterpret_cast<float *>(k_split + split_values(batch * hkv, nkb, D));
    auto *scores = reinterpret_cast<uint64_t *>(norm + (tasks + 3) / 4 * 4);
    const Means mq{mean, split, norm}, mk{mean + q_tasks * D, k_split, norm + q_tasks};
    constexpr int kWaves = kThreads / 64;
    block_mean_kernel<D><<<dim3(static_cast<unsigned>((tasks + kWaves - 1) / kWaves)), kThreads, 0, st>>>(
        q, k, static_cast<uint32_t>(q_tasks), static_cast<uint32_t>(tasks), mq, mk);
    const dim3 grid(static_cast<unsigned>(batch * hq * blocks_of(nqb, kTileQ)));
    const auto hq32 = static_cast<uint32_t>(hq), groups = static_cast<uint32_t>(hq / hkv);
    const int lq = static_cast<int>(q.len), lk = static_cast<int>(k.len);
#define TU_SELECT(BLOCKS)                                                                                              \
    block_choose_kernel<D, BLOCKS><<<grid, kChooseThreads<BLOCKS>, 0, st>>>(mq, mk, c, hq32, groups, nqb, nkb, lq, lk, \
                                                                            q.lengths, k.lengths, index)
    if (nkb <= 128) TU_SELECT(128);
    else if (nkb <= 512) TU_SELECT(512);
    else if (nkb <= 1024) TU_SELECT(1024);
    else if (nkb <= kMaxLdsBlocks) TU_SELECT(kMaxLdsBlocks);
    else {
        block_score_kernel<D><<<grid, kSelectThreads, 0, st>>>(mq.mean, mk.mean, c, hq32, groups, nqb, nkb, lq, lk,
                                                               q.lengths, k.lengths, scores);
        choose_kernel<<<dim3(static_cast<unsigned>((q_tasks + kWaves - 1) / kWaves)), kThreads, 0, st>>>(
            scores, c, hq32, nqb, nkb, static_cast<uint32_t>(q_tasks), lq, lk, q.lengths, k.lengths, index);
    }
#undef TU_SELECT
    return check_launch("tu_sage_block_select");
}

}  // namespace
}  // namespace tu

extern "C" int64_t tu_sage_block_select_workspace(int64_t batch, int64_t hq, int64_t hkv, int64_t lq, int64_t lk,
                                                  int64_t dim) {
    if (batch <= 0 || hq <= 0 || hkv <= 0 || lq <= 0 || lk <= 0 || dim <= 0) return 0;
    return tu::select_workspace(batch, hq, hkv, lq, lk, dim);
}

extern "C" int32_t tu_sage_block_select(const int8_t *q8, const float *q_scale, int64_t blkq, const int8_t *k8,
                                        const float *k_scale, int64_t blkk, int64_t batch, int64_t hq, int64_t hkv,
                                        int64_t lq, int64_t lk, int64_t dim, int64_t q_sb, int64_t q_sh, int64_t q_sl,
                                        int64_t k_sb, int64_t k_sh, int64_t k_sl, const int32_t *q_lengths,
                                        const int32_t *k_lengths, int64_t keep, int64_t sink_blocks,
                                        int64_t local_blocks, int32_t causal, void *workspace,
                                        int64_t workspace_bytes, int32_t *index, void *stream) {
    using namespace tu;
    TU_REQUIRE(dim == 64 || dim == 128, "block selection requires head_dim 64 or 128, got %lld",
               static_cast<long long>(dim));
    TU_REQUIRE(batch > 0 && hq > 0 && hkv > 0 && hq % hkv == 0, "block selection: hq must be a positive multiple of hkv");
    TU_REQUIRE(lq > 0 && lk > 0 && lq <= 0x7fffff00 && lk <= 0x7fffff00, "block selection: sequence lengths out of range");
    TU_REQUIRE(blkq > 0 && blkk > 0 && blkq <= 0x7fffffff && blkk <= 0x7fffffff, "block selection: scale blocks out of range");
    TU_REQUIRE(keep > 0 && sink_blocks >= 0 && local_blocks >= 0 && sink_blocks <= 0x3fffffff && local_blocks <= 0x3fffffff,
               "block selection: keep must be positive, sink and local blocks not negative");
    const int64_t nqb = blocks_of(lq, kQBlock), nkb = blocks_of(lk, kKBlock);
    TU_REQUIRE(batch * hq <= 65535 && batch * (hq * nqb + hkv * nkb) <= 0x7fffffff, "block selection grid too large");
    TU_REQUIRE(q8 && q_scale && k8 && k_scale && workspace && index, "block selection pointers must be non-null");
    TU_REQUIRE(q_sl % 16 == 0 && q_sh % 16 == 0 && q_sb % 16 == 0 && (reinterpret_cast<uintptr_t>(q8) & 15) == 0 &&
                   k_sl % 16 == 0 && k_sh % 16 == 0 && k_sb % 16 == 0 && (reinterpret_cast<uintptr_t>(k8) & 15) == 0,
               "block selection Q/K rows must be 16-byte aligned");
    const int64_t need = select_workspace(batch, hq, hkv, lq, lk, dim);
    TU_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= need,
               "block selection workspace must be 16-byte aligned and hold %lld bytes", static_cast<long long>(need));
    if (require_gfx950()) return -1;
    const Side q{q8, q_scale, q_lengths, q_sb, q_sh, q_sl, static_cast<uint32_t>(hq), static_cast<uint32_t>(lq),
                 static_cast<uint32_t>(blkq), static_cast<uint32_t>(blocks_of(lq, blkq)), static_cast<uint32_t>(nqb)};
    const Side k{k8, k_scale, k_lengths, k_sb, k_sh, k_sl, static_cast<uint32_t>(hkv), static_cast<uint32_t>(lk),
                 static_cast<uint32_t>(blkk), static_cast<uint32_t>(blocks_of(lk, blkk)), static_cast<uint32_t>(nkb)};
    const int64_t width = keep < nkb ? keep : nkb;
    const Choice c{static_cast<uint32_t>(width), static_cast<uint32_t>(sink_blocks), static_cast<uint32_t>(local_blocks),
                   static_cast<uint32_t>(width), causal != 0};
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dim == 128 ? launch_select<128>(q, k, batch, hq, hkv, c, workspace, index, st)
                      : launch_select<64>(q, k, batch, hq, hkv, c, workspace, index, st);
}
