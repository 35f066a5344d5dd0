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
// A choice between two near scores is right or wrong, so everything up to the
// choice is in 64 bits: code sums are integers, scale * sum is exact in fp64
// (24 + 15 bits), and the products run on v_mfma_f64_16x16x4_f64.  Two orders
// of these sums then differ by about 1e-15 of the score, where fp32 would
// change about one choice in a hundred thousand.
#include "tu_common.h"

namespace tu {
namespace {

typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int kQBlock = 128;  // rows of a query block
constexpr int kKBlock = 64;   // keys of a key block
constexpr int kThreads = 256;
constexpr int kSelectThreads = 512;
constexpr int kTileQ = 16;         // query blocks of a scoring workgroup (one MFMA's rows)
constexpr int kMaxLdsBlocks = 1024;  // key blocks whose keys fit LDS (16 rows of 8 KiB)

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
__device__ __forceinline__ void block_mean(const Side &s, uint32_t bh, uint32_t blk, double *__restrict__ mean,
                                           int lane) {
    constexpr int kLanesPerRow = D / 16;
    constexpr int kRpl = 64 / kLanesPerRow;  // rows per load
    constexpr int kLoads = kRows / kRpl;
    const uint32_t b = bh / s.heads, h = bh % s.heads;
    const int t0 = static_cast<int>(blk * kRows);
    const int valid = max(0, min(sample_end(s.lengths, b, static_cast<int>(s.len)) - t0, kRows));
    double *dst = mean + (static_cast<int64_t>(bh) * s.blocks + blk) * D;
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
            const double f = static_cast<double>(scale[static_cast<uint32_t>(row) / g]);
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
#pragma unroll
    for (int j = 0; j < (D == 128 ? 2 : 1); ++j) dst[c0 + j] = acc[j] / count;
}

// One wave per block: the query blocks first, then the key blocks.
template <int D>
__global__ __launch_bounds__(kThreads) void block_mean_kernel(Side q, Side k, uint32_t q_tasks, uint32_t tasks,
                                                              double *__restrict__ mean_q, double *__restrict__ mean_k) {
    const uint32_t task = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (task >= tasks) return;
    if (task < q_tasks) {
        block_mean<D, kQBlock>(q, task / q.blocks, task % q.blocks, mean_q, lane);
    } else {
        const uint32_t t = task - q_tasks;
        block_mean<D, kKBlock>(k, t / k.blocks, t % k.blocks, mean_k, lane);
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

__device__ __forceinline__ uint64_t forced_or(uint64_t key, int qb, int j, const Choice &c) {
    const int w = static_cast<int>(c.local);
    const bool near = w > 0 && j >= 2 * qb - (w - 1) && j <= 2 * qb + w;
    return near || j < static_cast<int>(c.sink) ? ~0ull : key;
}

// The `take` largest of the keys (key(p) is the lane's key of block 64 p +
// lane, 0 past the visible blocks and at least 1 in front), ties to the lower
// block, written in ascending order with -1 behind: the threshold is found bit
// by bit, counting keys at or above it, until a count fits.  kParts: keys of a
// lane, held in registers; 0: `parts` of them, read each time.
template <int kParts, typename Key>
__device__ __forceinline__ void select_row(int n, int take, int width, int lane, int parts, Key key,
                                           int32_t *__restrict__ out) {
    auto each = [&](auto visit) {
        if constexpr (kParts > 0) {
#pragma unroll
            for (int p = 0; p < kParts; ++p) visit(p);
        } else {
            for (int p = 0; p < parts; ++p) visit(p);
        }
    };
    uint64_t t = 1;
    if (take < n) {
        t = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t cand = t | 1ull << bit;
            int count = 0;
            each([&](int p) { count += __builtin_popcountll(__ballot(key(p) >= cand)); });
            if (count >= take) t = cand;
            if (count == take) break;
        }
    }
    int above = 0;
    each([&](int p) { above += __builtin_popcountll(__ballot(key(p) > t)); });
    const int allowed = take - above;
    const uint64_t below = (1ull << lane) - 1;
    int ties = 0, pos = 0;
    each([&](int p) {
        const uint64_t v = key(p);
        const uint64_t equal = __ballot(v == t);
        const bool chosen = v > t || (v == t && ties + __builtin_popcountll(equal & below) < allowed);
        const uint64_t mask = __ballot(chosen);
        if (chosen) out[pos + __builtin_popcountll(mask & below)] = 64 * p + lane;
        ties += __builtin_popcountll(equal);
        pos += __builtin_popcountll(mask);
    });
    for (int i = pos + lane; i < width; i += 64) out[i] = -1;
}

// Scores of 16 query blocks and all key blocks of one head, as ordered keys in
// LDS (kLds) or in `scores`, then (kLds) the choice, a wave per query block.
// The MFMA takes any order of the channels, so lane group g reads channels 8 u +
// 2 g and the next for the products 2 u and 2 u + 1: 64 bytes of a row per load
// (a quarter of the channels each, 256 bytes apart, fetched every line eight
// times: 85 us at 256 x 512 blocks of 40 heads).
template <int D, bool kLds, int kBlocks>
__global__ __launch_bounds__(kSelectThreads) void block_select_kernel(const double *__restrict__ mean_q,
                                                                const double *__restrict__ mean_k, Choice c,
                                                                uint32_t hq, uint32_t groups, uint32_t nqb,
                                                                uint32_t nkb, int lq, int lk,
                                                                const int32_t *__restrict__ q_len,
                                                                const int32_t *__restrict__ k_len,
                                                                uint64_t *__restrict__ scores,
                                                                int32_t *__restrict__ index) {
    __shared__ uint64_t keys[kLds ? kTileQ * kBlocks : 1];  // [query block][key block]
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
            const uint64_t key = j < visible_blocks(i, q_end, k_end, c.causal) ? forced_or(order_key(acc[r]), i, j, c) : 0;
            if constexpr (kLds) {
                if (j < kBlocks) keys[(4 * r + g) * kBlocks + j] = key;
            } else if (i < static_cast<int>(nqb) && j < static_cast<int>(nkb)) {
                scores[(static_cast<int64_t>(bh) * nqb + i) * nkb + j] = key;
            }
        }
    }
    if constexpr (kLds) {
        __syncthreads();
        for (int r = wave; r < kTileQ; r += kSelectThreads / 64) {
            const int i = i0 + r;
            if (i >= static_cast<int>(nqb)) break;
            const int n = visible_blocks(i, q_end, k_end, c.causal);
            int32_t *out = index + (static_cast<int64_t>(bh) * nqb + i) * c.width;
            uint64_t mine[kBlocks / 64];
#pragma unroll
            for (int p = 0; p < kBlocks / 64; ++p)
                mine[p] = 64 * p + lane < n ? keys[r * kBlocks + 64 * p + lane] : 0ull;
            select_row<kBlocks / 64>(n, min(static_cast<int>(c.keep), n), static_cast<int>(c.width), lane, 0,
                       [&](int p) { return mine[p]; }, out);
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
    select_row<0>(n, min(static_cast<int>(c.keep), n), static_cast<int>(c.width), lane, (n + 63) / 64,
               [&](int p) { return 64 * p + lane < n ? row[64 * p + lane] : 0ull; },
               index + static_cast<int64_t>(id) * c.width);
}

int64_t blocks_of(int64_t len, int64_t block) { return (len + block - 1) / block; }

// fp64 mean rows, then the ordered keys where they do not fit LDS.
int64_t select_workspace(int64_t batch, int64_t hq, int64_t hkv, int64_t lq, int64_t lk, int64_t dim) {
    const int64_t nqb = blocks_of(lq, kQBlock), nkb = blocks_of(lk, kKBlock);
    const int64_t means = batch * (hq * nqb + hkv * nkb) * dim;
    return (means + (nkb > kMaxLdsBlocks ? batch * hq * nqb * nkb : 0)) * 8;
}

template <int D>
int32_t launch_select(const Side &q, const Side &k, int64_t batch, int64_t hq, int64_t hkv, const Choice &c, void *ws,
                      int32_t *index, hipStream_t st) {
    const uint32_t nqb = q.blocks, nkb = k.blocks;
    const int64_t q_tasks = batch * hq * nqb, tasks = q_tasks + batch * hkv * nkb;
    auto *mean_q = static_cast<double *>(ws);
    double *mean_k = mean_q + q_tasks * D;
    auto *scores = reinterpret_cast<uint64_t *>(mean_k + batch * hkv * nkb * D);
    constexpr int kWaves = kThreads / 64;
    block_mean_kernel<D><<<dim3(static_cast<unsigned>((tasks + kWaves - 1) / kWaves)), kThreads, 0, st>>>(
        q, k, static_cast<uint32_t>(q_tasks), static_cast<uint32_t>(tasks), mean_q, mean_k);
    const dim3 grid(static_cast<unsigned>(batch * hq * blocks_of(nqb, kTileQ)));
#define TU_SELECT(LDS, BLOCKS)                                                                                          \
    block_select_kernel<D, LDS, BLOCKS><<<grid, kSelectThreads, 0, st>>>(                                                    \
        mean_q, mean_k, c, static_cast<uint32_t>(hq), static_cast<uint32_t>(hq / hkv), nqb, nkb, static_cast<int>(q.len), \
        static_cast<int>(k.len), q.lengths, k.lengths, scores, index)
    if (nkb <= 128) TU_SELECT(true, 128);
    else if (nkb <= 512) TU_SELECT(true, 512);
    else if (nkb <= kMaxLdsBlocks) TU_SELECT(true, kMaxLdsBlocks);
    else {
        TU_SELECT(false, 64);
        choose_kernel<<<dim3(static_cast<unsigned>((q_tasks + kWaves - 1) / kWaves)), kThreads, 0, st>>>(
            scores, c, static_cast<uint32_t>(hq), nqb, nkb, static_cast<uint32_t>(q_tasks), static_cast<int>(q.len),
            static_cast<int>(k.len), q.lengths, k.lengths, index);
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
