// Attention over the paged key/value cache in 8 bits (kv_cache.hip's pages).
// No counterpart in the reference's kernels.
//
//   out_r = sum_j p_rj v_j / sum_j p_rj over the keys j the row sees,
//   p = 2^(s - m), s = (q . k8) * (sm_scale * log2 e) * k_scale
// with q int8 codes and their scales, or 16-bit floats.  A float row is taken as
// integers of 16 bits, x ~ a (256 h + l) with h, l int8 and a = max |x| / 32512:
// two INT8 products in place of one in 16-bit floats, which would need every key
// converted.  An element is off by max |x| / 65024 at most, half a unit, whatever its
// own size: less than its own rounding where it is above 1/128 (bf16) or 1/16 (fp16)
// of the row's largest, more where it is below.
//
// Values are int8 codes with one scale a page.  They enter PV as fp16, exactly,
// and the page's scale enters the exponent: w = 2^(s + log2 v_scale - m') is about
// 2^7 for the largest p * v_scale of the row, so fp16 (11 bits, from 2^-14 on) holds
// the weights that matter, whatever the pages' scales are.  The row sum
// sum w / v_scale is kept apart, in fp32: of the unrounded w, or, where an MFMA adds
// up a tile's, of those that enter PV.
//   m' is held as the pair (score, log2 scale): far scores would swallow the
// scale in a sum.  Of a page whose log2 scale is less than the base's by more than
// 64, w may be no normal number where the page still matters in the row sum (its
// scores may be far above the base's): its weights are summed apart, as
// 2^(s - m' - log2 base scale).
//
// Two kernels: blocks of 16 rows (single tokens) read codes straight into registers;
// blocks of 128 or 256 share K and V tiles in LDS.  Both split a sequence's pages into
// ranges where the grid would leave the chip empty; a third merges.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_common.h"
#include "attn_plan.h"

namespace tu {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kPage = 64;
constexpr int kThreads = 256;
constexpr float kNoBase = -3.402823466e38f;  // score of a row's base before its first key
constexpr float kUp = 7.0f;                  // log2 of w at the base: fp16's room is used from 2^15 down to 2^-24
constexpr float kSlack = 8.0f;               // log2 of w above the base that moves it
constexpr float kLeastScale = -64.0f;        // log2 of a page's V scale, less the base's, below which its sum is taken apart
constexpr float kLeastRow = 1e-33f;          // a float row's units are made for at least this
constexpr float kFarMove = -100.0f;          // log2 of a factor that is taken in two steps
constexpr float kZeroValues = -90.0f;        // log2 V scale of a page whose values count as zeros
constexpr int kQInt8 = 2;                    // query types: 0 bf16, 1 fp16

struct CacheCall {
    const void *q;
    const float *q_scale;  // int8 queries: [batch][hq][nbq]
    uint32_t q_type, blkq, nbq;
    const int8_t *k_codes, *v_codes;
    const float *k_scale, *v_scale;
    const int32_t *table, *lengths, *q_lengths;
    int32_t width, pages;
    uint32_t batch, hkv, group;  // group: query heads of a K/V head
    uint32_t lq, rows;           // rows = lq * group, of one K/V head
    uint32_t row_blocks, parts;
    bool causal, out_fp16;
    float sm_log2;
    uint16_t *o;
    int64_t q_sb, q_sh, q_sl, o_sb, o_sh, o_sl;
    float *part_o, *part_m;  // [parts][batch * hkv * rows][D] and [..][4]: base score, base scale, sum
};

// A unit of work: rows of one K/V head over a range of its sequence's pages.
struct Unit {
    uint32_t b, hk, block, z;
    int n, length;   // query tokens and keys of the sequence
    int seen;        // keys that some row of the block sees
    int first, end;  // pages of the range
    int used;        // ranges that the block's pages fill
};

__device__ __forceinline__ int clamp_length(const int32_t *lengths, uint32_t b, int most) {
    return lengths ? min(max(lengths[b], 0), most) : most;
}

// Keys that query token `t` of n sees: all, or up to its own place, the n queries
// being the sequence's last tokens.
__device__ __forceinline__ int keys_of(const CacheCall &c, int t, int n, int length) {
    return c.causal ? min(length, max(length - n + t + 1, 0)) : length;
}

// Rows are numbered by token, then by head of the group.
template <int kRows>
__device__ __forceinline__ Unit unit_of(const CacheCall &c, uint32_t b, uint32_t hk, uint32_t block, uint32_t z) {
    Unit u;
    u.b = b, u.hk = hk, u.block = block, u.z = z;
    u.n = clamp_length(c.q_lengths, b, static_cast<int>(c.lq));
    u.length = clamp_length(c.lengths, b, c.width * kPage);
    const uint32_t last = min(c.rows, (block + 1) * kRows) - 1;
    const int token = min(static_cast<int>(last / c.group), u.n - 1);
    u.seen = block * kRows < static_cast<uint32_t>(u.n) * c.group ? keys_of(c, token, u.n, u.length) : 0;
    // (of the whole sequence: ranges of a causal call's blocks have one size)
    const int pages = (u.seen + kPage - 1) / kPage, per = ((u.length + kPage - 1) / kPage + c.parts - 1) / c.parts;
    u.first = min(pages, static_cast<int>(z) * per);
    u.end = min(pages, u.first + per);
    u.used = per ? (pages + per - 1) / per : 1;
    return u;
}

// Units by K/V head, so that the blocks of a head run on one XCD and its L2 reads
// the head's codes once.  Causal: blocks from the last, longest one on, heads
// fastest, so that the short ones fill the end.
template <int kRows>
__device__ __forceinline__ Unit unit_at(const CacheCall &c) {
    const uint32_t id = c.causal ? blockIdx.x : xcd_chunk(blockIdx.x, gridDim.x);
    uint32_t bh, block, z;
    if (c.causal) {
        const uint32_t heads = c.batch * c.hkv, rest = id / heads;
        bh = id % heads, z = rest % c.parts, block = c.row_blocks - 1 - rest / c.parts;
    } else {
        const uint32_t rest = id / c.parts;
        z = id % c.parts, block = rest % c.row_blocks, bh = rest / c.row_blocks;
    }
    return unit_of<kRows>(c, bh / c.hkv, bh % c.hkv, block, z);
}

// A row of the call: query token and head.  Rows past the last are the last.
struct Row {
    int token;
    uint32_t head;
};
__device__ __forceinline__ Row row_at(const CacheCall &c, uint32_t hk, uint32_t r) {
    r = min(r, c.rows - 1);
    return Row{static_cast<int>(r / c.group), hk * c.group + r % c.group};
}

// A lane's part of a query row, as it lies in memory: kSl pieces of 16 channels from
// `c0` on (c0 + step * i), and an int8 row's scale.
template <int kSl>
struct RowBits {
    u32x4 w[kSl][2];
    float scale;
};
template <int kSl, bool kTerms>
__device__ __forceinline__ RowBits<kSl> fetch_row(const CacheCall &c, const Row &row, uint32_t b, bool in, int c0, int step) {
    RowBits<kSl> r{};
    if (!in) return r;
    const int64_t off = b * c.q_sb + row.head * c.q_sh + row.token * c.q_sl + c0;
    if (!kTerms || c.q_type == kQInt8) {
#pragma unroll
        for (int i = 0; i < kSl; ++i) r.w[i][0] = *reinterpret_cast<const u32x4 *>(static_cast<const int8_t *>(c.q) + off + step * i);
        const int64_t at = static_cast<int64_t>(b * c.hkv * c.group + row.head) * c.nbq + static_cast<uint32_t>(row.token) / c.blkq;
        r.scale = c.q_scale[at];
    } else {
#pragma unroll
        for (int i = 0; i < kSl; ++i) {
            const auto *src = reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(c.q) + off + step * i);
            r.w[i][0] = src[0], r.w[i][1] = src[1];
        }
    }
    return r;
}

// An infinite scale as NaN: a score of minus infinity would leave a row without its key.
__device__ __forceinline__ float finite_or_nan(float scale) { return scale + (scale - scale); }

// The row as bytes h and l, and its factor (scale * sm_scale * log2 e of one unit of
// 256 h + l).  The row's lanes are the four groups of 16.
template <int kSl, bool kTerms>
__device__ __forceinline__ float row_codes(const CacheCall &c, const RowBits<kSl> &bits, i32x4 (&hi)[kSl], i32x4 (&lo)[kSl]) {
    if (!kTerms || c.q_type == kQInt8) {
#pragma unroll
        for (int i = 0; i < kSl; ++i) hi[i] = __builtin_bit_cast(i32x4, bits.w[i][0]), lo[i] = i32x4{0, 0, 0, 0};
        return finite_or_nan(bits.scale) * c.sm_log2 * (kTerms ? 0.00390625f : 1.0f);
    }
    float x[kSl][16];
#pragma unroll
    for (int i = 0; i < kSl; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const uint32_t pair = bits.w[i][e >> 3][(e >> 1) & 3], half = e & 1 ? pair >> 16 : pair & 0xffffu;
            x[i][e] = c.q_type == 0 ? bf16_bits_to_f32(half)
                                    : static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(half)));
        }
    // (bit patterns: a NaN is the largest)
    int top = 0;
#pragma unroll
    for (int i = 0; i < kSl; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max(top, static_cast<int>(__float_as_uint(x[i][e]) & 0x7fffffffu));
    top = xmax_i32(top);
    // (a NaN stays; of smaller rows the inverse would be infinite)
    const float amax = __int_as_float(max(top, __float_as_int(kLeastRow)));
    const float inverse = 32512.0f / amax;
#pragma unroll
    for (int i = 0; i < kSl; ++i) {
        hi[i] = lo[i] = i32x4{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int v = static_cast<int>(rintf(x[i][e] * inverse));
            const int h = (v + 128) >> 8, l = v - (h << 8);
            hi[i][e >> 2] |= (h & 0xff) << (8 * (e & 3));
            lo[i][e >> 2] |= (l & 0xff) << (8 * (e & 3));
        }
    }
    return finite_or_nan(amax) / 32512.0f * c.sm_log2;
}

// Four int8 codes as two pairs of fp16: the bytes biased by 128 below the
// exponent of 1024, less 1152.  With the selectors of zeros, four zeros.
struct Selectors {
    uint32_t low = 0x07010700u, high = 0x07030702u;
    __device__ __forceinline__ static Selectors of(bool zeros) {
        Selectors s;
        if (zeros) s.low = s.high = 0x07060706u;
        return s;
    }
};
__device__ __forceinline__ u32x2 codes_to_f16(uint32_t w, const Selectors &sel) {
    const f16x2_t bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    const uint32_t x = w ^ 0x80808080u;
    const uint32_t a = __builtin_amdgcn_perm(0x64806480u, x, sel.low);
    const uint32_t b = __builtin_amdgcn_perm(0x64806480u, x, sel.high);
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, a) - bias),
                 __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, b) - bias)};
}

__device__ __forceinline__ float lane_value(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

// Pages of a range, 64 at a time: lane i holds the i-th one's K and V planes' place
// in the pool, its K scale, log2 of the V scale and the V scale's inverse; a bit
// each: pages that are none (their place is the first's), and values of zero.
struct PageWindow {
    int at;
    float k_scale, v_log2, v_inverse;
    uint64_t none, zero;
    __device__ __forceinline__ void fetch(const CacheCall &c, const Unit &u, int from, int step, int lane) {
        int p = -1;
        if (from + step * lane < u.end) p = c.table[static_cast<int64_t>(u.b) * c.width + from + step * lane];
        const bool there = p >= 0 && p < c.pages;
        at = (there ? p : 0) * static_cast<int>(c.hkv) + static_cast<int>(u.hk);
        none = __ballot(!there);
        k_scale = c.k_scale[at];
        v_log2 = c.v_scale[at];
    }
    // What follows from the scales, which have landed then (here, and not in a loop that
    // uses them).  A NaN stays; below 2^-90, where a sum of weights over the scale might
    // be no number, the values count as zeros of that scale.
    __device__ __forceinline__ void landed() {
        const float v = v_log2;
        zero = __ballot(v <= 8.077935669e-28f);
        v_log2 = v <= 8.077935669e-28f ? kZeroValues : __builtin_amdgcn_logf(v);
        v_inverse = v <= 8.077935669e-28f ? 1.2379400392853803e27f : __builtin_amdgcn_rcpf(v);
        k_scale = finite_or_nan(k_scale);
        asm volatile("" : "+v"(k_scale));
    }
    __device__ __forceinline__ int64_t place(int i) const { return __builtin_amdgcn_readlane(at, i); }
    __device__ __forceinline__ bool there(int i) const { return !(none >> i & 1); }
    __device__ __forceinline__ bool zeros(int i) const { return zero >> i & 1; }
};

// The softmax state of a row: base (score, log2 of a V scale), and in the lane
// its share of the sum of w / v_scale.
struct RowState {
    float m = kNoBase, v = 0.0f, l = 0.0f;
    // Of a page far below the base's scale, w / v_scale of score x: at most 2^(kSlack + kUp
    // - kZeroValues), as the base has not moved.
    __device__ __forceinline__ float apart(float x) const { return __builtin_amdgcn_exp2f((x - m) + (kUp - v)); }
};

// Results of a unit's rows: o[ds][r] = channel 16 ds + 4 g + r of the row of the
// lane's column, l its whole sum.  Written out, or for the merge.
template <int D>
__device__ __forceinline__ void store_row(const CacheCall &c, const Unit &u, const f32x4 (&o)[D / 16], float m, float v, float l,
                                          uint32_t r, int g) {
    const Row row = row_at(c, u.hk, r);
    if (u.used > 1) {
        if (r >= c.rows) return;
        const int64_t rows = static_cast<int64_t>(c.batch) * c.hkv * c.rows;
        const int64_t at = u.z * rows + static_cast<int64_t>(u.b * c.hkv + u.hk) * c.rows + r;
#pragma unroll
        for (int ds = 0; ds < D / 16; ++ds) *reinterpret_cast<f32x4 *>(c.part_o + at * D + 16 * ds + 4 * g) = o[ds];
        if (g == 0) *reinterpret_cast<f32x4 *>(c.part_m + at * 4) = f32x4{m, v, l, 0.0f};
        return;
    }
    // (a sum of 0 is a row that saw no key; one that is NaN stays NaN)
    const bool some = l != 0.0f && row.token < u.n;
    const float inv = 1.0f / l;
    uint16_t *op = c.o + u.b * c.o_sb + row.head * c.o_sh + row.token * c.o_sl;
#pragma unroll
    for (int ds = 0; ds < D / 16; ds += 2) {
        uint32_t w[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x4 a = o[ds + i] * inv;
            const uint32_t p0 = c.out_fp16 ? hw_f16x2_bits(a[0], a[1]) : hw_bf16x2_bits(a[0], a[1]);
            const uint32_t p1 = c.out_fp16 ? hw_f16x2_bits(a[2], a[3]) : hw_bf16x2_bits(a[2], a[3]);
            w[i][0] = some ? p0 : 0;
            w[i][1] = some ? p1 : 0;
        }
        // each lane ends with 8 contiguous channels of one row
        auto lo = __builtin_amdgcn_permlane16_swap(w[0][0], w[1][0], false, false);
        auto hi = __builtin_amdgcn_permlane16_swap(w[0][1], w[1][1], false, false);
        if (r >= c.rows) continue;
        auto *dst = reinterpret_cast<u32x2 *>(op + 16 * (ds + (g & 1)) + 8 * (g >> 1));
        dst[0] = u32x2{lo[0], hi[0]};
        dst[1] = u32x2{lo[1], hi[1]};
    }
}

// to + l * 2^a, given 2^a.  A sum over V scales may lie as far above 1 as 2^a lies below
// fp32's range (a base of scale 2^-30 left for one of 2^100): two steps then.
__device__ __forceinline__ float moved(float l, float a, float power, float to = 0.0f) {
    float sum = __builtin_fmaf(power, l, to);
    if (__any(a < kFarMove)) {
        const float half = __builtin_amdgcn_exp2f(0.5f * a);
        if (a < kFarMove) sum = to + (l * half) * half;
    }
    return sum;
}

// The other of two bases where it is higher: by score, and log2 of the V scale.
__device__ __forceinline__ bool higher(float m, float v, float than_m, float than_v) {
    return (m - than_m) + (v - than_v) > 0.0f;
}

// ---------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------
// A workgroup of four waves has 16 rows of one K/V head (more rows: more workgroups,
// whose codes come from L2 but for the first); its waves take the pages of the unit's
// range in turn, each for itself, and are merged at the end.  A wave reads a page's
// codes straight into the MFMA operands: keys 16 g + e of a page belong to lane group
// g throughout, so that a lane's 16 bytes of a V^T row are the keys whose weights it
// holds, and a key row's bytes go to the lanes in runs of D / 4.  The next page's
// loads (16 KiB a wave at D = 128) are in flight while one is computed: what a CU
// needs to keep HBM busy.
constexpr int kFewRows = 16;
template <int D>
struct PageRegs {
    i32x4 k[4][D / 64];
    u32x4 v[D / 16];
    __device__ __forceinline__ void load(const CacheCall &c, int64_t at, int g, int lc) {
        const int8_t *k_page = c.k_codes + at * kPage * D, *v_page = c.v_codes + at * kPage * D;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < D / 64; ++i)
                k[t][i] = *reinterpret_cast<const i32x4 *>(k_page + (16 * (lc >> 2) + 4 * t + (lc & 3)) * D + D / 4 * g + 16 * i);
#pragma unroll
        for (int ds = 0; ds < D / 16; ++ds)
            v[ds] = *reinterpret_cast<const u32x4 *>(v_page + (16 * ds + lc) * kPage + 16 * g);
    }
};

template <int D>
__global__ __launch_bounds__(kThreads, 2) void cache_few_kernel(CacheCall c) {
    constexpr int kSl = D / 64, kDS = D / 16;
    __shared__ __align__(16) float merge_o[3][kDS][64][4];
    __shared__ float merge_m[4][64][3];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, lc = lane & 15;
    const Unit u = unit_at<kFewRows>(c);
    if (u.z > 0 && static_cast<int>(u.z) >= u.used) return;  // the whole workgroup: nothing is left for the range
    // The loads of a start, in an order that leaves three in a row (length; rows and
    // table; codes and scales): one token of 32 heads over 4000, 12.3 -> 11.4 us.
    const uint32_t r = u.block * kFewRows + lc;
    const Row row = row_at(c, u.hk, r);
    const bool in = r < c.rows && row.token < u.n;
    const RowBits<kSl> bits = fetch_row<kSl, true>(c, row, u.b, in, D / 4 * g, 16);
    PageWindow window;
    int base = u.first + wave;  // page of the window's lane 0; the wave's pages are 4 apart
    window.fetch(c, u, base, 4, lane);
    auto place = [&](int p) {  // of page p of the sequence, one of the window's
        return window.place((p - base) >> 2);
    };
    PageRegs<D> even, odd;
    int p = base;
    if (p < u.end) even.load(c, place(p), g, lc);
    i32x4 qh[kSl], ql[kSl];
    const float factor = row_codes<kSl, true>(c, bits, qh, ql);
    window.landed();
    const int limit = in ? keys_of(c, row.token, u.n, u.length) : 0;
    RowState st;
    f32x4 o[kDS];
#pragma unroll
    for (int ds = 0; ds < kDS; ++ds) o[ds] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    auto compute = [&](const PageRegs<D> &r, int p) {
        const int at = (p - base) >> 2;
        const bool there = window.there(at);
        const float k_scale = lane_value(window.k_scale, at), v_log2 = lane_value(window.v_log2, at);
        const int key0 = p * kPage + 16 * g;  // the lane's keys are key0 ..+15
        i32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            i32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < kSl; ++i) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(r.k[t][i], qh[i], acc, 0, 0, 0);
            acc <<= 8;
#pragma unroll
            for (int i = 0; i < kSl; ++i) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(r.k[t][i], ql[i], acc, 0, 0, 0);
            s[t] = acc;
        }
        const float f = factor * k_scale;
        const int seen = there ? limit - key0 : 0;  // the first so many of the lane's keys
        float x[16], top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            x[e] = static_cast<float>(s[e >> 2][e & 3]) * f;
            if (e < seen) top = fmaxf(top, x[e]);
        }
        const bool need = (top - st.m) + (v_log2 - st.v) > kSlack;
        if (__any(need)) {
            // a row's base moves by its own scores alone
            const float row_top = xmax_f32(top);
            if ((row_top - st.m) + (v_log2 - st.v) > kSlack) {
                const float a = (st.m - row_top) + (st.v - v_log2), alpha = __builtin_amdgcn_exp2f(a);
                st.m = row_top, st.v = v_log2;
                st.l = moved(st.l, a, alpha);
#pragma unroll
                for (int ds = 0; ds < kDS; ++ds) o[ds] *= alpha;
            }
        }
        const float d = v_log2 - st.v;
        float sum = 0.0f;
        f16x8 w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 packed;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float y[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int e = 8 * h + 2 * j + i;
                    y[i] = e < seen ? __builtin_amdgcn_exp2f((x[e] - st.m) + (d + kUp)) : 0.0f;
                    sum += y[i];
                }
                packed[j] = hw_f16x2_bits(y[0], y[1]);
            }
            w[h] = __builtin_bit_cast(f16x8, packed);
        }
        // w / v_scale, the scale being 2^(base's + d) (a lane without keys has no part in a NaN)
        float inverse = __builtin_amdgcn_exp2f(-(st.v + d));
        if (__any(d < kLeastScale)) {
            float apart = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) apart += e < seen ? st.apart(x[e]) : 0.0f;
            if (d < kLeastScale) sum = apart, inverse = 1.0f;
        }
        if (seen > 0) st.l = __builtin_fmaf(sum, inverse, st.l);
        if (window.zeros(at)) return;
#pragma unroll
        for (int ds = 0; ds < kDS; ++ds) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x2 a = codes_to_f16(r.v[ds][2 * h], Selectors{}), b = codes_to_f16(r.v[ds][2 * h + 1], Selectors{});
                const f16x8 v = __builtin_bit_cast(f16x8, (u32x4{a[0], a[1], b[0], b[1]}));
                o[ds] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[h], o[ds], 0, 0, 0);
            }
        }
    };

    // Two pages a step, so that the registers of one are filled while the other is computed.
#pragma clang loop unroll(disable)
    for (; p < u.end; p += 8) {
        if (p + 4 < u.end) odd.load(c, place(p + 4), g, lc);
        compute(even, p);
        if (p + 4 >= u.end) break;
        const bool refill = p + 8 - base >= 64 * 4;
        if (!refill && p + 8 < u.end) even.load(c, place(p + 8), g, lc);
        compute(odd, p + 4);
        if (refill && p + 8 < u.end) {
            base = p + 8;
            window.fetch(c, u, base, 4, lane);
            window.landed();
            even.load(c, place(p + 8), g, lc);
        }
    }

    // The waves' states, merged by the first.
    st.l = xsum_f32(st.l);
    if (u.end - u.first > 1) {
        merge_m[wave][lane][0] = st.m;
        merge_m[wave][lane][1] = st.v;
        merge_m[wave][lane][2] = st.l;
        if (wave > 0) {
#pragma unroll
            for (int ds = 0; ds < kDS; ++ds) *reinterpret_cast<f32x4 *>(merge_o[wave - 1][ds][lane]) = o[ds];
        }
        __syncthreads();
    }
    if (wave > 0) return;
    if (u.end - u.first > 1) {
        float m = st.m, v = st.v;
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            const float mi = merge_m[i][lane][0], vi = merge_m[i][lane][1];
            if (merge_m[i][lane][2] != 0.0f && higher(mi, vi, m, v)) m = mi, v = vi;
        }
        float l = 0.0f;
        f32x4 sum[kDS] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float li = merge_m[i][lane][2];
            if (li == 0.0f) continue;  // saw nothing
            const float a = (merge_m[i][lane][0] - m) + (merge_m[i][lane][1] - v), wi = __builtin_amdgcn_exp2f(a);
            l = moved(li, a, wi, l);
#pragma unroll
            for (int ds = 0; ds < kDS; ++ds) {
                const f32x4 x = i == 0 ? o[ds] : *reinterpret_cast<const f32x4 *>(merge_o[i - (i > 0)][ds][lane]);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[ds][e] = __builtin_fmaf(wi, x[e], sum[ds][e]);
            }
        }
        st.m = m, st.v = v, st.l = l;
#pragma unroll
        for (int ds = 0; ds < kDS; ++ds) o[ds] = sum[ds];
    }
    store_row<D>(c, u, o, st.m, st.v, st.l, r, g);
}

// ---------------------------------------------------------------------------
// Many rows
// ---------------------------------------------------------------------------
// A workgroup has 128 or 256 rows of one K/V head: one or two groups of four waves,
// 32 rows a wave.  Two groups of 128 share a CU either way; within one workgroup they
// share the tiles too (half the reads from L2 and conversions of V), and run opposite
// each other: one's MFMAs beside the other's softmax.  Pages stream through LDS: keys
// as codes by direct-to-LDS loads, a ring of four; values through registers, converted
// to fp16 once, a ring of two.
//   Bound by issue: a step of 256 rows takes 3300 cycles at D = 128 (1.4 us at 2.36
// GHz), 48 of its 52 MFMAs a wave with their LDS reads and the softmax alone, in the
// same phases, 2310 of them, on one box.  The other 30 % are loads, conversions of V and
// waits; without them the card lowers its clock (random operands: 2.0 GHz, 1.17 us a
// step).  4680 rows x 32760 keys, 40 heads, int8 queries: 2.15-2.26 ms, box to box,
// 1390-1460 TFLOP/s (one group: 2.45 ms).
constexpr int kQT = 2;           // 16-row fragments of a wave
constexpr int kWaveRows = 16 * kQT;
constexpr int kGroupRows = 4 * kWaveRows;
constexpr int kKRing = 4;
constexpr float kSummed = -1.0f;

template <int D>
struct Tiles {
    static constexpr int kK = kPage * D;      // bytes of a K stage
    static constexpr int kV = kPage * D * 2;  // of a V stage
    static constexpr int kV0 = kKRing * kK;
    static constexpr int kBytes = kV0 + 2 * kV;
};

// LDS row of a K tile -> key: within each half of 32, row 16 t + i holds key
// 8 (i >> 2) + 4 t + (i & 3), so that a lane group owns 8 contiguous keys of a
// half, one 16-byte piece of a V^T row.
__device__ __forceinline__ int key_of_row(int row) {
    return (row & ~31) + 8 * ((row & 15) >> 2) + 4 * ((row >> 4) & 1) + (row & 3);
}

// Loads of 1 KiB that a wave of kWaves has of a page's keys, and of its values (the
// first waves only, where there are more waves than loads).
template <int D, int kWaves>
constexpr int kPieces = Tiles<D>::kK / 1024 >= kWaves ? Tiles<D>::kK / 1024 / kWaves : 1;

template <int D, int kWaves>
struct ManyGeom {
    uint32_t k_src[kPieces<D, kWaves>];  // a lane's 16 bytes of a page's keys
    uint32_t k_rd[D / 64];               // operand of QK^T
    uint32_t v_rd[2];                    // operand of PV, half 0 / 1
    uint32_t v_wr[2];                    // where the two halves of a lane's 16 values go
    static constexpr bool kAll = Tiles<D>::kK / 1024 >= kWaves;
    bool loads;                          // whether the wave loads (kAll: every one does)
};

// 16-byte pieces of a row are XORed with row bits, so that 16 lanes that read
// one column of 16 rows meet distinct banks, and so do lanes that write V^T.
__device__ __forceinline__ int v_swizzle(int ch) { return ((ch >> 1) & 7) ^ (ch & 1); }
template <int D, int kWaves>
__device__ __forceinline__ ManyGeom<D, kWaves> many_geom(int wave, int lane) {
    ManyGeom<D, kWaves> gm;
    const int g = lane >> 4, lc = lane & 15;
    gm.loads = wave < Tiles<D>::kK / 1024;
#pragma unroll
    for (int i = 0; i < kPieces<D, kWaves>; ++i) {
        const int piece = (kPieces<D, kWaves> * wave + i) * 64 + lane;  // of 16 bytes in LDS
        const int row = piece / (D / 16), at = piece % (D / 16);
        const int swizzle = D == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
        gm.k_src[i] = static_cast<uint32_t>(key_of_row(row) * D + (at ^ swizzle) * 16);
    }
    const int ch = wave * 16 + lane / 4;
#pragma unroll
    for (int e = 0; e < 2; ++e) gm.v_wr[e] = static_cast<uint32_t>(ch * 128 + (((2 * (lane % 4) + e) ^ v_swizzle(ch)) << 4));
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
        gm.k_rd[i] = static_cast<uint32_t>(lc * D + (D == 128 ? ((4 * i + g) ^ ((lc >> 1) & 7)) : (g ^ ((lc >> 2) & 3))) * 16);
#pragma unroll
    for (int i = 0; i < 2; ++i) gm.v_rd[i] = static_cast<uint32_t>(lc * 128 + (((4 * i + g) ^ v_swizzle(lc)) << 4));
    return gm;
}

// Bases of the wave's rows.  Where every base is small in size (`ready`), a base
// is also held as one number, base = m + v - kUp.
template <int D>
struct ManyState {
    RowState row[kQT];
    float base[kQT];
    f32x4 o[D / 16][kQT];
    // of the wave:
    float m_most;  // largest |m|; infinite while a row has seen no key
    float v_most;  // largest v
    __device__ __forceinline__ void init() {
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) {
            base[qt] = kNoBase;
#pragma unroll
            for (int ds = 0; ds < D / 16; ++ds) o[ds][qt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        m_most = INFINITY, v_most = 0.0f;
    }
    // Moves the bases of rows that a page's scores pass by more than kSlack; top:
    // each lane's largest.  A row's base moves by its own scores alone.
    __device__ __forceinline__ void move(const float (&top)[kQT], float v_log2) {
        float size = 0.0f, v = kZeroValues;
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) {
            const float row_top = xmax_f32(top[qt]);
            const bool go = (row_top - row[qt].m) + (v_log2 - row[qt].v) > kSlack;
            const float a = go ? (row[qt].m - row_top) + (row[qt].v - v_log2) : 0.0f, alpha = __builtin_amdgcn_exp2f(a);
            row[qt].m = go ? row_top : row[qt].m;
            row[qt].v = go ? v_log2 : row[qt].v;
            row[qt].l = moved(row[qt].l, a, alpha);
#pragma unroll
            for (int ds = 0; ds < D / 16; ++ds) o[ds][qt] *= alpha;
            base[qt] = (row[qt].m + row[qt].v) - kUp;
            size = fmaxf(size, fabsf(row[qt].m));
            v = fmaxf(v, row[qt].v);
        }
#pragma unroll
        for (int i = 1; i < 16; i <<= 1) {
            size = fmaxf(size, __shfl_xor(size, i));
            v = fmaxf(v, __shfl_xor(v, i));
        }
        m_most = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(size)));
        v_most = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
    }
};

// S^T of a tile from its K fragments: s[t][qt][r] = key 32 (t >> 1) + 8 g + 4 (t &
// 1) + r, row 16 qt + lc.  One term: biased (kBias); two: the integer 256 q_h . k +
// q_l . k.
template <int D, bool kTerms>
__device__ __forceinline__ void many_qk(const i32x4 (&kf)[4][D / 64], const i32x4 (&qh)[kQT][D / 64],
                                        const i32x4 (&ql)[kQT][D / 64], i32x4 (&s)[4][kQT]) {
    constexpr int kSl = D / 64;
    constexpr int kFrom = kTerms ? 0 : kBias;
    i32x4 z[4][kQT];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt)
            z[t][qt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t][0], qh[qt][0], i32x4{kFrom, kFrom, kFrom, kFrom}, 0, 0, 0);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) {
            if constexpr (D == 128) z[t][qt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t][kSl - 1], qh[qt][kSl - 1], z[t][qt], 0, 0, 0);
            s[t][qt] = z[t][qt];
        }
    if constexpr (kTerms) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int qt = 0; qt < kQT; ++qt) {
                i32x4 acc = s[t][qt] << 8;
#pragma unroll
                for (int i = 0; i < kSl; ++i) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t][i], ql[qt][i], acc, 0, 0, 0);
                s[t][qt] = acc;
            }
    }
}

// The lane's largest score of a tile, an integer as many_qk leaves it.
__device__ __forceinline__ int tile_top(const i32x4 (&s)[4][kQT], int qt) {
    int mi = imax3(s[0][qt][0], s[0][qt][1], s[0][qt][2]);
    mi = imax3(mi, s[0][qt][3], s[1][qt][0]);
    mi = imax3(mi, s[1][qt][1], s[1][qt][2]);
    mi = imax3(mi, s[1][qt][3], s[2][qt][0]);
    mi = imax3(mi, s[2][qt][1], s[2][qt][2]);
    mi = imax3(mi, s[2][qt][3], s[3][qt][0]);
    mi = imax3(mi, s[3][qt][1], s[3][qt][2]);
    return max(mi, s[3][qt][3]);
}

template <bool kTerms>
__device__ __forceinline__ float score(int s) {
    return kTerms ? static_cast<float>(s) : __int_as_float(s) - kBiasF;
}

// Weights w[h][qt] of a tile (keys 32 h + 8 g ..+7) in the careful form: for rows
// that see a part of it (keys from `seen[qt]` on take no part), for scores whose
// size would swallow fractions in a sum, and for pages whose V scale is far below
// the base's, where weights too small for fp16 still count in the sum.  The product
// is rounded as the base was, and the sum of weights is one of 32 bits, here.
template <int D, bool kTerms>
__device__ __forceinline__ void careful_weights(i32x4 (&s)[4][kQT], const float (&f)[kQT], float v_log2, const int (&seen)[kQT],
                                                int g, ManyState<D> &st, f16x8 (&w)[2][kQT]) {
    constexpr int kLeast = static_cast<int>(0x80000000u);
    float top[kQT];
    bool need = false;
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
        const int t0 = seen[qt] - 1 - 8 * g;  // key 8 g + c is seen iff c <= t0
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int hidden = (t0 - (32 * (t >> 1) + 4 * (t & 1) + r)) >> 31;
                s[t][qt][r] = (s[t][qt][r] & ~hidden) | (kLeast & hidden);
            }
        const int mi = tile_top(s, qt);
        top[qt] = mi == kLeast ? -INFINITY : score<kTerms>(mi) * f[qt];
        need = need || (top[qt] - st.row[qt].m) + (v_log2 - st.row[qt].v) > kSlack;
    }
    if (__any(need)) st.move(top, v_log2);
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
        const int t0 = seen[qt] - 1 - 8 * g;
        const float d = v_log2 - st.row[qt].v;
        float sum = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 packed;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float y[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int e = 2 * j + i;  // key 32 h + 8 g + e
                    const int hidden = (t0 - (32 * h + e)) >> 31;
                    const float x = (score<kTerms>(s[2 * h + (e >> 2)][qt][e & 3]) * f[qt] - st.row[qt].m) + (d + kUp);
                    y[i] = __int_as_float(__float_as_int(__builtin_amdgcn_exp2f(x)) & ~hidden);
                    sum += y[i];
                }
                packed[j] = hw_f16x2_bits(y[0], y[1]);
            }
            w[h][qt] = __builtin_bit_cast(f16x8, packed);
        }
        float inverse = __builtin_amdgcn_exp2f(-(st.row[qt].v + d));
        if (__any(d < kLeastScale)) {
            float apart = 0.0f;
#pragma unroll
            for (int c = 0; c < 16; ++c) {  // key 32 (c >> 3) + 8 g + (c & 7)
                const int hidden = (t0 - (32 * (c >> 3) + (c & 7))) >> 31;
                const float x = score<kTerms>(s[c >> 2][qt][c & 3]) * f[qt];
                apart += __int_as_float(__float_as_int(st.row[qt].apart(x)) & ~hidden);
            }
            if (d < kLeastScale) sum = apart, inverse = 1.0f;
        }
        // (a row that sees nothing of the tile has no part in a NaN)
        const float all = xsum_f32(sum);
        if (seen[qt] > 0) st.row[qt].l = __builtin_fmaf(all, inverse, st.row[qt].l);
    }
}

// Softmax of a tile that every row of the wave sees whole.  Weights are
// fma(score, f, c) with c = log2 v_scale - base, less than 2^12 in size and so exact
// to 2^-13 (with the bias of the integer scores in it where that keeps it there),
// and are summed, as fp16, by an MFMA beside PV's.  Returns what that sum is to be
// multiplied by: 1 / v_scale, or kSummed where the careful form has summed.
template <int D, bool kTerms>
__device__ __forceinline__ float whole_weights(i32x4 (&s)[4][kQT], const float (&f)[kQT], float f_most, float v_log2,
                                               float v_inverse, int g, ManyState<D> &st, f16x8 (&w)[2][kQT]) {
    float top[kQT];
    bool need = false;
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
        top[qt] = score<kTerms>(tile_top(s, qt)) * f[qt];
        need = need || (top[qt] + v_log2) - st.base[qt] > kSlack + kUp;
    }
    if (__any(need)) st.move(top, v_log2);
    if (__builtin_expect(!(st.m_most < 4000.0f && v_log2 >= st.v_most - 8.0f), 0)) {
        const int seen[kQT] = {kPage, kPage};
        careful_weights<D, kTerms>(s, f, v_log2, seen, g, st, w);
        return kSummed;
    }
    auto weights = [&](auto folded_tag) __attribute__((always_inline)) {
        constexpr bool kFolded = decltype(folded_tag)::value;
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) {
            const float c = v_log2 - (kFolded ? __builtin_fmaf(kBiasF, f[qt], st.base[qt]) : st.base[qt]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 packed;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float y[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int e = 2 * j + i;  // key 32 h + 8 g + e
                        const int si = s[2 * h + (e >> 2)][qt][e & 3];
                        const float x = kFolded ? __int_as_float(si) : score<kTerms>(si);
                        y[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, f[qt], c));
                    }
                    packed[j] = hw_f16x2_bits(y[0], y[1]);
                }
                w[h][qt] = __builtin_bit_cast(f16x8, packed);
            }
        }
    };
    if constexpr (kTerms) {
        weights(std::false_type{});
    } else {
        if (__builtin_fmaf(kBiasF, f_most, st.m_most) < 4000.0f) weights(std::true_type{});
        else weights(std::false_type{});
    }
    return v_inverse;
}

// O^T += V^T w and the sum of the tile's weights, times `inverse` (see whole_weights).
template <int D, int kWaves>
__device__ __forceinline__ void many_pv(const int8_t *stage, const ManyGeom<D, kWaves> &gm, const f16x8 (&w)[2][kQT], const f16x8 &ones,
                                        float inverse, ManyState<D> &st) {
    f32x4 sum[kQT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        f16x8 vf[D / 16];
#pragma unroll
        for (int ds = 0; ds < D / 16; ++ds) vf[ds] = *reinterpret_cast<const f16x8 *>(stage + gm.v_rd[h] + ds * 16 * 128);
#pragma unroll
        for (int ds = 0; ds < D / 16; ++ds)
#pragma unroll
            for (int qt = 0; qt < kQT; ++qt)
                st.o[ds][qt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[ds], w[h][qt], st.o[ds][qt], 0, 0, 0);
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt)
            sum[qt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, w[h][qt], h ? sum[qt] : f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
    }
    if (!(inverse < 0.0f)) {
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) st.row[qt].l = __builtin_fmaf(sum[qt][0], inverse, st.row[qt].l);
    }
}

// A steady step's MFMAs: QK^T of one page, PV of the page before it.
template <int D, bool kTerms, int kWaves>
__device__ __forceinline__ void many_cluster(const int8_t *k_stage, const int8_t *v_stage, const ManyGeom<D, kWaves> &gm,
                                             const i32x4 (&qh)[kQT][D / 64], const i32x4 (&ql)[kQT][D / 64],
                                             i32x4 (&s)[4][kQT], const f16x8 (&w)[2][kQT], const f16x8 &ones,
                                             float inverse, ManyState<D> &st) {
    constexpr int kSl = D / 64;
    // (over the other workgroup's softmax on the same SIMD)
    __builtin_amdgcn_s_setprio(3);
    i32x4 kf[4][kSl];
#pragma unroll
    for (int i = 0; i < kSl; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) kf[t][i] = *reinterpret_cast<const i32x4 *>(k_stage + gm.k_rd[i] + t * 16 * D);
    many_qk<D, kTerms>(kf, qh, ql, s);
    many_pv<D>(v_stage, gm, w, ones, inverse, st);
    // Issue order, with at most 16 LDS reads in flight: the K reads, the first
    // products, half of the V^T reads, products, the other half, the rest.
    constexpr int kK = 4 * kSl, kV = D / 16, kQk = kK * kQT * (kTerms ? 2 : 1), kPv = 2 * kQT * (kV + 1);
    __builtin_amdgcn_sched_group_barrier(0x100, kK, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, kK, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, kV, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, kQk - kK + kPv / 9, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, kV, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, kPv - kPv / 9, 0);
    __builtin_amdgcn_s_setprio(0);
}

// A page's keys into a ring stage; its values into registers, and from there into one.
// (One overload for each, as the host's pass takes no template of the load.)
#define TU_MANY_LOAD_K(D, WAVES)                                                                                       \
    __device__ __forceinline__ void many_load_k(int8_t *stage, __amdgpu_buffer_rsrc_t rs, const ManyGeom<D, WAVES> &gm,  \
                                                int wave) {                                                            \
        constexpr int kN = kPieces<D, WAVES>;                                                                          \
        _Pragma("unroll") for (int i = 0; i < kN; ++i)                                                                 \
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void *)(stage + (kN * wave + i) * 1024), 16, gm.k_src[i], 0, 0, 0); \
    }
TU_MANY_LOAD_K(128, 4)
TU_MANY_LOAD_K(64, 4)
TU_MANY_LOAD_K(128, 8)
TU_MANY_LOAD_K(64, 8)
#undef TU_MANY_LOAD_K

// The compiler would wait for every load in flight before a write to LDS, as loads of
// keys write there too (never to these places); so the writes are spelled out, and
// the wait for them stands before the barrier that hands them over.
__device__ __forceinline__ void write_lds(uint32_t at, u32x4 x) {
    asm volatile("ds_write_b128 %0, %1" ::"v"(at), "v"(x) : "memory");
}
template <int D, int kWaves>
__device__ __forceinline__ void many_store_v(uint32_t stage, const ManyGeom<D, kWaves> &gm, const u32x4 (&v)[kPieces<D, kWaves>],
                                             const Selectors &sel) {
#pragma unroll
    for (int i = 0; i < kPieces<D, kWaves>; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const u32x2 a = codes_to_f16(v[i][2 * e], sel), b = codes_to_f16(v[i][2 * e + 1], sel);
            write_lds(stage + gm.v_wr[e] + i * (16 * kWaves * 128), u32x4{a[0], a[1], b[0], b[1]});
        }
}

// Four waves at D = 64 with one term leave the registers for a third workgroup on a CU
// (8192 x 4096, 12 heads: 134 -> 115 us; with two terms they spill, and it gains nothing).
template <int D, bool kTerms, int kGroups>
__global__ __launch_bounds__(256 * kGroups, kGroups == 2 ? 1 : D == 64 && !kTerms ? 3 : 2) void cache_many_kernel(CacheCall call) {
    constexpr int kSl = D / 64, kDS = D / 16, kWaves = 4 * kGroups, kLoads = kPieces<D, kWaves>, kRows = kGroupRows * kGroups;
    __shared__ __align__(1024) int8_t lds[Tiles<D>::kBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, lc = lane & 15;
    const int group = wave >> 2;
    const Unit u = unit_at<kRows>(call);
    if (u.z > 0 && static_cast<int>(u.z) >= u.used) return;  // the whole workgroup: nothing is left for the range
    const uint32_t row0 = u.block * kRows + wave * kWaveRows;
    auto row_of = [&](int qt) { return row_at(call, u.hk, row0 + 16 * qt + lc); };
    // (as few rows' start: three loads in a row; the first pages' are on their way while
    // the rows are taken apart)
    RowBits<kSl> bits[kQT];
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
        const Row row = row_of(qt);
        bits[qt] = fetch_row<kSl, kTerms>(call, row, u.b, row0 + 16 * qt + lc < call.rows && row.token < u.n, 16 * g, 64);
    }
    PageWindow window;
    int base = u.first;
    window.fetch(call, u, base, 1, lane);
    const ManyGeom<D, kWaves> gm = many_geom<D, kWaves>(wave, lane);

    f16x8 ones;
#pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = static_cast<_Float16>(1.0f);
    const int8_t *k_codes = call.k_codes, *v_codes = call.v_codes;
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) int8_t *)lds));

    i32x4 s[4][kQT];
    f16x8 w[2][kQT];
    float inverse = kSummed;  // of the page whose weights w holds
    u32x4 v[2][kLoads];  // values of the next two pages, by parity
    auto at_of = [&](int p) { return min(p, u.end - 1) - base; };
    auto place = [&](int p) { return window.place(at_of(p)); };
    auto k_stage = [&](int p) { return lds + (p - u.first) % kKRing * Tiles<D>::kK; };
    auto v_stage = [&](int p) { return lds + Tiles<D>::kV0 + (p - u.first) % 2 * Tiles<D>::kV; };
    auto load_k = [&](int8_t *stage, int64_t at) __attribute__((always_inline)) {
        if (gm.kAll || gm.loads) many_load_k(stage, make_rsrc(k_codes + at * kPage * D, kPage * D), gm, wave);
    };
    auto load_v = [&](u32x4 (&v)[kLoads], int64_t at) __attribute__((always_inline)) {
        const int8_t *page = v_codes + at * kPage * D;
        if (!gm.kAll && !gm.loads) return;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) v[i] = *reinterpret_cast<const u32x4 *>(page + (i * 64 * kWaves + threadIdx.x) * 16);
    };
    if (u.first < u.end) {
        load_v(v[0], place(u.first));
        load_k(k_stage(u.first), place(u.first));
        load_k(k_stage(u.first + 1), place(u.first + 1));
        load_v(v[1], place(u.first + 1));
    }

    i32x4 qh[kQT][kSl], ql[kQT][kSl];
    float factor[kQT];
    int limit[kQT];
    ManyState<D> st;
    st.init();
    float most = 0.0f;
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
        factor[qt] = row_codes<kSl, kTerms>(call, bits[qt], qh[qt], ql[qt]);
        limit[qt] = keys_of(call, min(row_of(qt).token, max(u.n - 1, 0)), u.n, u.length);
        most = fmaxf(most, factor[qt]);
    }
#pragma unroll
    for (int i = 1; i < 16; i <<= 1) most = fmaxf(most, __shfl_xor(most, i));
    const float factor_most = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(most)));
    // pages that all rows of the wave see whole: those of its first row
    const int whole = __builtin_amdgcn_readfirstlane(
        keys_of(call, min(row_at(call, u.hk, row0).token, max(u.n - 1, 0)), u.n, u.length) / kPage);
    window.landed();

    auto store_v = [&](int parity, const u32x4 (&v)[kLoads], int p) __attribute__((always_inline)) {
        if (gm.kAll || gm.loads)
            many_store_v<D>(lds_at + Tiles<D>::kV0 + parity * Tiles<D>::kV, gm, v, Selectors::of(window.zeros(p - base)));
    };
    auto softmax_part = [&](int p) __attribute__((always_inline)) {
        const int at = p - base;
        const float k_scale = lane_value(window.k_scale, at), v_log2 = lane_value(window.v_log2, at);
        const bool there = window.there(at);
        float f[kQT];
        int seen[kQT];
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) f[qt] = factor[qt] * k_scale, seen[qt] = there ? limit[qt] - p * kPage : 0;
        careful_weights<D, kTerms>(s, f, v_log2, seen, g, st, w);
        inverse = kSummed;
    };
    auto softmax_whole = [&](int p) __attribute__((always_inline)) {
        const int at = p - base;
        const float k_scale = lane_value(window.k_scale, at), v_log2 = lane_value(window.v_log2, at);
        float f[kQT];
#pragma unroll
        for (int qt = 0; qt < kQT; ++qt) f[qt] = factor[qt] * k_scale;
        inverse = whole_weights<D, kTerms>(s, f, factor_most * k_scale, v_log2, lane_value(window.v_inverse, at), g, st, w);
    };
    auto qk = [&](int p) __attribute__((always_inline)) {
        i32x4 kf[4][kSl];
#pragma unroll
        for (int i = 0; i < kSl; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) kf[t][i] = *reinterpret_cast<const i32x4 *>(k_stage(p) + gm.k_rd[i] + t * 16 * D);
        many_qk<D, kTerms>(kf, qh, ql, s);
    };

    // Step p: QK^T of page p + 1 and PV of page p, then the softmax of page p + 1.
    // Interval p, between two barriers, has for group 0 step p, and for group 1 the
    // softmax of page p and the MFMAs of step p: the groups' MFMAs and softmaxes stand
    // opposite each other on a SIMD.  In interval p keys of p + 1 and values of p are
    // read from LDS, values of p + 1 converted into the stage that interval p - 1 read
    // last, and keys of p + 3 and values of p + 3 (into the registers that those of p +
    // 1 left) loaded: each load has two intervals to land.
    constexpr std::integral_constant<int, 0> kEven;
    constexpr std::integral_constant<int, 1> kOdd;
    auto landed = [&] __attribute__((always_inline)) {
        // the keys that the next interval reads: all but this one's loads and the
        // values loaded behind them
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(3 * kLoads));
        __builtin_amdgcn_s_waitcnt(lgkmcnt_imm(0));
        wg_barrier();
    };
    if (u.first < u.end) {
        store_v(0, v[0], u.first);
        load_k(k_stage(u.first + 2), place(u.first + 2));
        load_v(v[0], place(u.first + 2));
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        qk(u.first);
        if (kGroups == 1 || group == 0) softmax_part(u.first);
        if (kGroups == 2) wg_barrier();
        if (kGroups == 2 && group == 1) softmax_part(u.first);
        for (int p = u.first; p < u.end;) {
            if (p + 3 - base >= 64 && base + 64 < u.end) {
                base = p;
                window.fetch(call, u, base, 1, lane);
                window.landed();
            }
            // steps whose next page every row sees whole: up to the first that is none,
            // and as far as the window reaches three pages on
            const uint64_t none = window.none & (p + 1 - base < 64 ? ~0ull << (p + 1 - base) : 0);
            int to = min(min(u.end, whole) - 1, base + 64 < u.end ? base + 61 : u.end);
            if (none) to = min(to, base + static_cast<int>(__builtin_ctzll(none)) - 1);
            // the loads of interval p, and the values it converts
            auto feed = [&](auto parity_tag, int8_t *k_to) __attribute__((always_inline)) {
                constexpr int kParity = decltype(parity_tag)::value;
                store_v(kParity ^ 1, v[kParity ^ 1], min(p + 1, u.end - 1));
                const int64_t next = place(p + 3);
                load_k(k_to, next);
                __builtin_amdgcn_sched_barrier(0);  // (the wait before the barrier counts on the order)
                load_v(v[kParity ^ 1], next);
            };
            if (p < to) {
                int k1 = (p + 1 - u.first) % kKRing * Tiles<D>::kK;
                auto step = [&](auto parity_tag) __attribute__((always_inline)) {
                    constexpr int kParity = decltype(parity_tag)::value;
                    many_cluster<D, kTerms>(lds + k1, lds + Tiles<D>::kV0 + kParity * Tiles<D>::kV, gm, qh, ql, s, w, ones, inverse, st);
                    feed(parity_tag, lds + (k1 + 2 * Tiles<D>::kK) % (kKRing * Tiles<D>::kK));
                    if (kGroups == 2 && group == 1) landed();
                    softmax_whole(p + 1);
                    k1 = (k1 + Tiles<D>::kK) % (kKRing * Tiles<D>::kK);
                    ++p;
                    if (kGroups == 1 || group == 0) landed();
                };
                // (without it the compiler's waits inside would be for other ways to here)
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
                if ((p - u.first) % 2) step(kOdd);
#pragma clang loop unroll(disable)
                while (p + 1 < to) {
                    step(kEven);
                    step(kOdd);
                }
                if (p < to) step(kEven);
            }
            if (p + 3 - base >= 64 && base + 64 < u.end) continue;  // the window's end
            // One step of another kind: a page that some row sees in part, or the last.
            if (p + 1 < u.end) qk(p + 1);
            if ((p - u.first) % 2) feed(kOdd, k_stage(p + 3));
            else feed(kEven, k_stage(p + 3));
            many_pv<D>(v_stage(p), gm, w, ones, inverse, st);
            if (kGroups == 2 && group == 1) landed();
            if (p + 1 < u.end) softmax_part(p + 1);
            if (kGroups == 1 || group == 0) landed();
            ++p;
        }
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // (loads past the range's end into LDS)
    }
    // (the call's fields are read again, not kept through the loop)
    auto *again = (const CacheCall *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(again));
    const CacheCall c = *again;
#pragma unroll
    for (int qt = 0; qt < kQT; ++qt) {
        f32x4 o[kDS];
#pragma unroll
        for (int ds = 0; ds < kDS; ++ds) o[ds] = st.o[ds][qt];
        store_row<D>(c, u, o, st.row[qt].m, st.row[qt].v, st.row[qt].l, row0 + 16 * qt + lc, g);
    }
}

// ---------------------------------------------------------------------------
// The merge
// ---------------------------------------------------------------------------
// A row's ranges: D / 8 threads for each, 8 channels a thread.  A range that saw
// none of the row's keys has a sum of 0 and is left out; a NaN stays.  With few rows
// a call has too few threads for one to walk a row's ranges (32 of them took 9.2 us
// at 64 rows, D = 128): a workgroup has one row then, and kTurns = kThreads / (D / 8)
// ranges at a time.
struct MergeState {
    float m = kNoBase, v = 0.0f, l = 0.0f, acc[8] = {};
    // kN ranges' states (m, v, l) and 8 channels of their sums
    template <int kN>
    __device__ __forceinline__ void add(const f32x4 (&x)[kN], const f32x4 (&a)[kN], const f32x4 (&b)[kN], int there) {
        float m_new = m, v_new = v;
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (i < there && x[i][2] != 0.0f && higher(x[i][0], x[i][1], m_new, v_new)) m_new = x[i][0], v_new = x[i][1];
        const float l_old = l, a_old = l == 0.0f ? 0.0f : (m - m_new) + (v - v_new);
        const float old = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(a_old);
        m = m_new, v = v_new;
        l *= old;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = old == 0.0f ? 0.0f : acc[e] * old;
        float least = a_old;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if (i >= there || x[i][2] == 0.0f) continue;
            const float ai = (x[i][0] - m) + (x[i][1] - v), wi = __builtin_amdgcn_exp2f(ai);
            least = fminf(least, ai);
            l = __builtin_fmaf(wi, x[i][2], l);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[e] = __builtin_fmaf(wi, a[i][e], acc[e]);
                acc[4 + e] = __builtin_fmaf(wi, b[i][e], acc[4 + e]);
            }
        }
        if (!__any(least < kFarMove)) return;
        l = moved(l_old, a_old, old);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if (i >= there || x[i][2] == 0.0f) continue;
            const float ai = (x[i][0] - m) + (x[i][1] - v);
            l = moved(x[i][2], ai, __builtin_amdgcn_exp2f(ai), l);
        }
    }
};

template <int D, int kRows, int kTurns>
__global__ __launch_bounds__(kThreads) void cache_merge_kernel(CacheCall c) {
    constexpr int kTpr = D / 8;
    const int64_t rows = static_cast<int64_t>(c.batch) * c.hkv * c.rows;
    const int turn = kTurns > 1 ? threadIdx.x / kTpr : 0;
    const int64_t at = kTurns > 1 ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * (kThreads / kTpr) + threadIdx.x / kTpr;
    if (at >= rows) return;
    const uint32_t bh = static_cast<uint32_t>(at / c.rows), r = static_cast<uint32_t>(at % c.rows);
    const int d0 = (threadIdx.x % kTpr) * 8;
    constexpr int kAhead = kTurns > 1 ? 2 : 4;  // ranges whose loads are in flight together
    f32x4 x[kAhead], a[kAhead], b[kAhead];
    auto load = [&](int z0, int last) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t from = min(z0 + i * kTurns, last) * rows + at;
            x[i] = *reinterpret_cast<const f32x4 *>(c.part_m + from * 4);
            a[i] = *reinterpret_cast<const f32x4 *>(c.part_o + from * D + d0);
            b[i] = *reinterpret_cast<const f32x4 *>(c.part_o + from * D + d0 + 4);
        }
    };
    // (of few rows before the length is here, ranges that nothing fills among them)
    if (kTurns > 1) load(turn, static_cast<int>(c.parts) - 1);
    const Unit u = unit_of<kRows>(c, bh / c.hkv, bh % c.hkv, r / kRows, 0);
    if (u.used <= 1) return;
    const Row row = row_at(c, u.hk, r);
    MergeState st;
    for (int z0 = turn; z0 < u.used; z0 += kAhead * kTurns) {
        if (kTurns == 1 || z0 > turn) load(z0, u.used - 1);
        st.add(x, a, b, (u.used - z0 + kTurns - 1) / kTurns);
    }
    if constexpr (kTurns > 1) {
        __shared__ __align__(16) f32x4 all[3][kTurns][kTpr];
        all[0][turn][threadIdx.x % kTpr] = f32x4{st.m, st.v, st.l, 0.0f};
        all[1][turn][threadIdx.x % kTpr] = f32x4{st.acc[0], st.acc[1], st.acc[2], st.acc[3]};
        all[2][turn][threadIdx.x % kTpr] = f32x4{st.acc[4], st.acc[5], st.acc[6], st.acc[7]};
        __syncthreads();
        if (turn > 0) return;
        constexpr int kStep = 4;
#pragma unroll
        for (int t = 1; t < kTurns; t += kStep) {
            f32x4 xs[kStep], as[kStep], bs[kStep];
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                const int from = min(t + i, kTurns - 1);
                xs[i] = all[0][from][threadIdx.x], as[i] = all[1][from][threadIdx.x], bs[i] = all[2][from][threadIdx.x];
            }
            st.add(xs, as, bs, kTurns - t);
        }
    }
    const bool some = st.l != 0.0f && row.token < u.n;
    const float inv = 1.0f / st.l;
    u32x4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float p = st.acc[2 * e] * inv, q = st.acc[2 * e + 1] * inv;
        out[e] = some ? (c.out_fp16 ? hw_f16x2_bits(p, q) : hw_bf16x2_bits(p, q)) : 0;
    }
    auto *dst = reinterpret_cast<u32x2 *>(c.o + u.b * c.o_sb + row.head * c.o_sh + row.token * c.o_sl + d0);
    dst[0] = u32x2{out[0], out[1]};
    dst[1] = u32x2{out[2], out[3]};
}

// ---------------------------------------------------------------------------
// The plan
// ---------------------------------------------------------------------------
struct CachePlan {
    int32_t rows;  // of a row block: kFewRows, or 128 or 256 (many)
    uint32_t row_blocks, parts;
};

// What a block of rows costs, in steps of a page at 256 rows (1.4 us at D = 128): a step
// on a CU that has one, two or three of its workgroups (as many as `places`), and the
// pages that a start and an end take as long as.  Fitted at D = 128; D = 64 takes the
// same ratios.
struct BlockCost {
    int32_t rows;
    int64_t places;
    double step[3], start;
};
constexpr BlockCost kFewCost = {kFewRows, 2, {0.28, 0.575, 0.0}, 7.0};
constexpr BlockCost kManyCost = {kGroupRows, 2, {0.78, 1.08, 1.4}, 4.0};
constexpr BlockCost kTwoGroupsCost = {2 * kGroupRows, 1, {1.0, 0.0, 0.0}, 4.0};

// Time of a launch: its rounds of the places there are, and a merge: 3 steps and its
// bytes, 7 MB a step (at 256 CUs).
//   Measured, us, blocks of 16 / 128 rows, each at its best number of ranges: 64 rows of
// 8 K/V heads x 8192 keys 18 / 27, 256 rows 37 / 34, 64 rows of 40 heads x 2048 19 / 24,
// 64 of 128 heads 34 / 36, 77 of 12 heads x 513 at D = 64 7.2 / 13.  One round more is
// dear: one row of 40 heads x 131040, 12 ranges 235, 13 319; and one workgroup a CU reads
// as fast as two (one row of 256 heads x 8190: 1 range 82, 2 ranges 87).
//   128 / 256 rows: 4680 rows x 32760 keys, 40 heads, int8 queries 2450 / 2240; 1560 x
// 9360, 12 heads, by ranges: 1: 184 / 214, 2: 133 / 125, 3: 99 / 97, 4: 120 / 133, 6:
// 111 / 111; 8192 x 4096 at D = 64, 12 heads: 115 / 147.
//   Causal: empty ranges of early blocks end at once, and long blocks go first.
// 4001 x 4001, 2 x 16 heads: 1 range 143, 2 ranges 224; 2050 x 6000 at D = 64, 18
// heads, 128 rows a block: 123, 87.
double launch_cost(const BlockCost &b, int64_t units, int64_t parts, int64_t per, double share, bool causal, double part_bytes,
                   int64_t cus) {
    const int64_t slots = b.places * cus;
    auto step = [&](double n) { return n <= 0.0 ? 0.0 : n <= cus ? b.step[0] : n <= 2 * cus ? b.step[1] : b.step[2]; };
    const double n = static_cast<double>(units * parts) * share, full = n / static_cast<double>(slots);
    double steps = step(n);
    if (full > 1.0) {
        const int64_t rounds = units * parts / slots;
        steps = causal ? (full + 0.5) * step(slots)
                       : static_cast<double>(rounds) * step(slots) + step(static_cast<double>(units * parts - rounds * slots));
    }
    const double merge = parts > 1 ? 3.0 + static_cast<double>(parts) * part_bytes * 2.0 / (7e6 * static_cast<double>(cus) / 256.0) : 0.0;
    return steps * (static_cast<double>(per) + b.start) + merge;
}

CachePlan cache_plan(int64_t batch, int64_t hkv, int64_t lq, int64_t group, int64_t dim, int64_t pages, bool int8, bool causal,
                     int64_t cus, int64_t max_bytes) {
    const int64_t rows = lq * group;
    const int64_t row_bytes = batch * hkv * rows * (dim + 4) * static_cast<int64_t>(sizeof(float));
    // of a causal call's keys, the part that its mean row sees
    const double tokens = static_cast<double>(pages * kPage);
    const double share = causal ? std::max(0.5, 1.0 - 0.5 * static_cast<double>(lq) / tokens) : 1.0;
    CachePlan best{};
    double best_cost = 0.0;
    auto consider = [&](const BlockCost &b) {
        const int64_t blocks = (rows + b.rows - 1) / b.rows, units = batch * hkv * blocks;
        // (a page for each wave of few rows, two pages of many)
        const int64_t most = std::min<int64_t>(max_bytes / row_bytes, b.rows == kFewRows ? std::min<int64_t>((pages + 3) / 4, 256)
                                                                                         : std::min<int64_t>(pages / 2, 64));
        for (int64_t parts = 1;;) {
            const int64_t per = (pages + parts - 1) / parts;
            const double cost = launch_cost(b, units, parts, per, share, causal, static_cast<double>(row_bytes), cus);
            if (!best.rows || cost < best_cost) {
                best = CachePlan{b.rows, static_cast<uint32_t>(blocks), static_cast<uint32_t>(parts)};
                best_cost = cost;
            }
            if (per == 1 || units * parts > 3 * b.places * cus) break;
            parts = (pages + per - 2) / (per - 1);  // the next number of ranges that are shorter
            if (parts > most) break;
        }
    };
    consider(kFewCost);
    if (rows > kFewRows) {
        BlockCost many = kManyCost;
        if (dim == 64 && int8) many.places = 3;
        consider(many);
        consider(kTwoGroupsCost);
    }
    return best;
}

// Sizes that the plan's and the kernels' arithmetic holds.
bool cache_sizes(int64_t batch, int64_t hq, int64_t hkv, int64_t lq, int64_t max_length, int64_t cus) {
    return batch > 0 && batch <= 65535 && hkv > 0 && hq >= hkv && hq <= 65535 && lq > 0 && lq <= 0x7fffff00 &&
           lq * (hq / hkv) <= 0x7fffff00 && batch * hkv * (lq * (hq / hkv)) <= int64_t{0x7fffffff} * 16 && max_length > 0 && cus > 0 &&
           cus <= 65535;
}

int64_t cache_workspace(const CachePlan &p, int64_t batch, int64_t hkv, int64_t rows, int64_t dim) {
    return p.parts > 1 ? p.parts * batch * hkv * rows * (dim + 4) * static_cast<int64_t>(sizeof(float)) : 0;
}

// The plan of a call with all the workspace it wants; no rows for bad sizes.
CachePlan whole_plan(int64_t batch, int64_t hq, int64_t hkv, int64_t lq, int64_t dim, int64_t max_length, int32_t q_type,
                     int32_t causal, int32_t cus) {
    if (!cache_sizes(batch, hq, hkv, lq, max_length, cus) || (dim != 64 && dim != 128)) return CachePlan{};
    const int64_t pages = std::min<int64_t>((max_length - 1) / kPage + 1, 0x7fffffff / kPage - 1);
    return cache_plan(batch, hkv, lq, hq / hkv, dim, pages, q_type == kQInt8, causal != 0, cus, INT64_MAX);
}

}  // namespace
}  // namespace tu

extern "C" int64_t tu_kv_cache_attn_workspace(int64_t batch, int64_t hq, int64_t hkv, int64_t lq, int64_t dim, int64_t max_length,
                                              int32_t q_type, int32_t causal, int32_t cus) {
    const tu::CachePlan plan = tu::whole_plan(batch, hq, hkv, lq, dim, max_length, q_type, causal, cus);
    return plan.rows ? tu::cache_workspace(plan, batch, hkv, lq * (hq / hkv), dim) : 0;
}

extern "C" int32_t tu_kv_cache_attn_plan(int64_t batch, int64_t hq, int64_t hkv, int64_t lq, int64_t dim, int64_t max_length,
                                         int32_t q_type, int32_t causal, int32_t cus) {
    const tu::CachePlan plan = tu::whole_plan(batch, hq, hkv, lq, dim, max_length, q_type, causal, cus);
    return plan.rows << 16 | static_cast<int32_t>(plan.parts);
}

extern "C" int32_t tu_kv_cache_attn(const void *q, const float *q_scale, int32_t q_type, int64_t blkq, const int8_t *k_codes,
                                    const int8_t *v_codes, const float *k_scale, const float *v_scale, int64_t pages,
                                    const int32_t *block_table, int64_t width, const int32_t *lengths,
                                    const int32_t *q_lengths, void *o, int64_t batch, int64_t hq, int64_t hkv, int64_t lq,
                                    int64_t dim, int64_t q_sb, int64_t q_sh, int64_t q_sl, int64_t o_sb, int64_t o_sh,
                                    int64_t o_sl, float sm_scale, int32_t causal, int64_t max_length, int32_t cus,
                                    void *workspace, int64_t workspace_bytes, void *stream) {
    using namespace tu;
    TU_REQUIRE(dim == 64 || dim == 128, "cache attention requires head_dim 64 or 128, got %lld", static_cast<long long>(dim));
    TU_REQUIRE(q_type >= 0 && q_type <= kQInt8, "cache attention query type must be 0 (bf16), 1 (fp16) or 2 (int8), got %d", q_type);
    TU_REQUIRE(batch > 0 && hq > 0 && hkv > 0 && hq % hkv == 0, "cache attention: hq must be a positive multiple of hkv");
    TU_REQUIRE(cache_sizes(batch, hq, hkv, lq, max_length, cus), "cache attention sizes out of range");
    TU_REQUIRE(width > 0 && width <= 0x7fffffff / kPage - 1 && pages > 0 && pages <= 0x7fffffff,
               "cache attention block table or page count out of range");
    TU_REQUIRE(pages * hkv <= 0x7fffffff, "cache attention: pages of all heads out of range");
    TU_REQUIRE(q && k_codes && v_codes && k_scale && v_scale && block_table && lengths && o && (q_scale || q_type != kQInt8),
               "cache attention pointers must be non-null");
    TU_REQUIRE(q_type != kQInt8 || (blkq > 0 && blkq <= 0x7fffffff), "cache attention needs blkq > 0");
    TU_REQUIRE(sm_scale > 0.0f && std::isfinite(sm_scale * kLog2e), "cache attention sm_scale must be positive and finite");
    const int64_t piece = q_type == kQInt8 ? 16 : 8;
    TU_REQUIRE(q_sb % piece == 0 && q_sh % piece == 0 && q_sl % piece == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0,
               "cache attention query rows must be 16-byte aligned");
    TU_REQUIRE((reinterpret_cast<uintptr_t>(k_codes) & 15) == 0 && (reinterpret_cast<uintptr_t>(v_codes) & 15) == 0 &&
                   o_sb % 4 == 0 && o_sh % 4 == 0 && o_sl % 4 == 0 && (reinterpret_cast<uintptr_t>(o) & 7) == 0,
               "cache attention codes and output must be aligned");
    TU_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "cache attention workspace must be 16-byte aligned");
    const int64_t rows = lq * (hq / hkv);
    const CachePlan plan = cache_plan(batch, hkv, lq, hq / hkv, dim, std::min<int64_t>((max_length - 1) / kPage + 1, width),
                                      q_type == kQInt8, causal != 0, cus, workspace ? workspace_bytes : 0);
    const int64_t units = batch * hkv * plan.row_blocks * plan.parts;
    // a launch's threads are counted in 32 bits (a merge has no more workgroups than a row each)
    constexpr int64_t kMost = 0xffffffff;
    TU_REQUIRE(units <= kMost / (plan.rows == 2 * kGroupRows ? 512 : 256) &&
                   (plan.parts == 1 || batch * hkv * rows <= kMost / kThreads),
               "cache attention grid too large");
    if (require_gfx950()) return -1;
    CacheCall c{};
    c.q = q, c.q_scale = q_scale, c.q_type = static_cast<uint32_t>(q_type);
    c.blkq = q_type == kQInt8 ? static_cast<uint32_t>(blkq) : 1;
    c.nbq = q_type == kQInt8 ? static_cast<uint32_t>((lq + blkq - 1) / blkq) : 0;
    c.k_codes = k_codes, c.v_codes = v_codes, c.k_scale = k_scale, c.v_scale = v_scale;
    c.table = block_table, c.lengths = lengths, c.q_lengths = q_lengths;
    c.width = static_cast<int32_t>(width), c.pages = static_cast<int32_t>(pages);
    c.batch = static_cast<uint32_t>(batch), c.hkv = static_cast<uint32_t>(hkv), c.group = static_cast<uint32_t>(hq / hkv);
    c.lq = static_cast<uint32_t>(lq), c.rows = static_cast<uint32_t>(rows);
    c.row_blocks = plan.row_blocks, c.parts = plan.parts;
    c.causal = causal != 0, c.out_fp16 = q_type == 1;
    c.sm_log2 = sm_scale * kLog2e;
    c.o = static_cast<uint16_t *>(o);
    c.q_sb = q_sb, c.q_sh = q_sh, c.q_sl = q_sl, c.o_sb = o_sb, c.o_sh = o_sh, c.o_sl = o_sl;
    c.part_o = static_cast<float *>(workspace);
    c.part_m = c.part_o + plan.parts * batch * hkv * rows * dim;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(units));
    // (the merge of many rows: one thread walks a row's few ranges)
#define TU_CACHE_MERGE(D, ROWS, TURNS)                                                                                 \
    do {                                                                                                               \
        constexpr int64_t kRowsPerWg = TURNS > 1 ? 1 : kThreads / (D / 8);                                             \
        const dim3 merge(static_cast<unsigned>((batch * hkv * rows + kRowsPerWg - 1) / kRowsPerWg));                   \
        if (plan.parts > 1) cache_merge_kernel<D, ROWS, TURNS><<<merge, kThreads, 0, s>>>(c);                          \
    } while (0)
#define TU_CACHE_ATTN(D)                                                                                               \
    do {                                                                                                               \
        if (plan.rows == kFewRows) {                                                                                   \
            cache_few_kernel<D><<<grid, kThreads, 0, s>>>(c);                                                          \
            TU_CACHE_MERGE(D, kFewRows, kThreads / (D / 8));                                                           \
        } else if (plan.rows == 128) {                                                                                 \
            if (q_type == kQInt8) cache_many_kernel<D, false, 1><<<grid, 256, 0, s>>>(c);                              \
            else cache_many_kernel<D, true, 1><<<grid, 256, 0, s>>>(c);                                                \
            TU_CACHE_MERGE(D, 128, 1);                                                                                 \
        } else {                                                                                                       \
            if (q_type == kQInt8) cache_many_kernel<D, false, 2><<<grid, 512, 0, s>>>(c);                              \
            else cache_many_kernel<D, true, 2><<<grid, 512, 0, s>>>(c);                                                \
            TU_CACHE_MERGE(D, 256, 1);                                                                                 \
        }                                                                                                              \
    } while (0)
    if (dim == 128) TU_CACHE_ATTN(128);
    else TU_CACHE_ATTN(64);
#undef TU_CACHE_ATTN
#undef TU_CACHE_MERGE
    return check_launch("tu_kv_cache_attn");
}
