// A paged key/value cache in 8 bits: new tokens are quantized as they are
// written, and read back.  No counterpart in the reference's kernels.
//
// A page holds 64 tokens of every K/V head, with one scale a head for its keys
// and one for its values:
//   key codes int8 [page][head][64][D], value codes int8 [page][head][D][64]
// (the tiles that cache_attn.hip reads: K rows for QK^T, V^T for PV).
//
// Writing tokens into a page, K and V apart:
//   s  = max(s of the tokens in the page before, max |new x| / 127, 1e-7 / 127)
//   code = rint(x * (1 / s)) in fp32, |code| <= 127
// and where s grew, the earlier tokens' codes become rint((code * s_before) *
// (1 / s)).  A page belongs to one workgroup, so nothing is shared; codes behind
// the last new token keep their bytes.  The maximum is one of bit patterns, so
// that a NaN or infinite x makes the scale one, and the page's codes 0.
//
// Bound by HBM where much is written or read (2 bytes of a 16-bit type and 1 of codes
// an element): 32760 tokens of 40 heads, D = 128, are written and read in about 200 us
// each, 5 TB/s, the rate of a large copy.  By a chain of four loads (length, page, row,
// scale) for single tokens: 32 tokens of 8 heads in 5.8 us.
//   Heads come fastest in the grid, so that workgroups that run together read whole
// rows of a tensor with tokens first (a token for 32 sequences and back: 14 -> 12 us;
// tensors with heads first lose 2 percent).  Each load and store of a wave covers
// whole lines, V^T by way of LDS (487 -> 401 us for 32760 tokens and back).
#include <algorithm>

#include "tu_common.h"

namespace tu {
namespace {

constexpr int kPage = 64;
constexpr int kThreads = 256;
constexpr int64_t kMostWgs = 0xffffffff / kThreads;  // a launch's threads are counted in 32 bits

// Where a call's tokens lie in the pages.
struct Pages {
    const int32_t *table;    // [batch][width]
    const int32_t *lengths;  // [batch]
    int32_t width;           // pages of a sequence
    int32_t count;           // pages of the pool
    uint32_t hkv;
};

__device__ __forceinline__ int held(const Pages &p, uint32_t b) { return min(max(p.lengths[b], 0), p.width * kPage); }

// A block's page, or -1 where the table names none.
__device__ __forceinline__ int page_of(const Pages &p, uint32_t b, int block) {
    if (block >= p.width) return -1;
    const int page = p.table[static_cast<int64_t>(b) * p.width + block];
    return page >= 0 && page < p.count ? page : -1;
}

template <int kType>
__device__ __forceinline__ float element(uint32_t pair, int half) {
    const uint32_t bits = half ? pair >> 16 : pair & 0xffffu;
    if constexpr (kType == 0) return bf16_bits_to_f32(bits);
    else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Signed byte e of a dword.
__device__ __forceinline__ float byte_of(uint32_t w, int e) {
    return static_cast<float>(static_cast<int8_t>(w >> (8 * e)));
}

// The largest bit pattern of the workgroup's threads.
__device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t *part) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), off)));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return max(max(part[0], part[1]), max(part[2], part[3]));
}

// Scale of a page from the largest |x| of its new tokens, and what codes are made with.
struct Quantizer {
    float scale, inverse, before;
    bool grown;
    __device__ __forceinline__ Quantizer(uint32_t amax, float scale_before, bool any_before) {
        const float fresh = __uint_as_float(max(amax, __float_as_uint(1e-7f))) / 127.0f;
        before = any_before ? fabsf(scale_before) : 0.0f;
        const uint32_t bits = max(magnitude(fresh), magnitude(before));
        scale = __uint_as_float(bits);
        grown = any_before && bits != magnitude(before);
        // (an infinite or NaN scale: every code 0)
        inverse = bits < 0x7f800000u ? 1.0f / scale : 0.0f;
    }
    __device__ __forceinline__ uint32_t code(float x) const {
        const float c = rintf(x * inverse);
        // infinity * 0 is a NaN, whose code is 0 as well
        return static_cast<uint32_t>(c == c ? static_cast<int>(fminf(fmaxf(c, -127.0f), 127.0f)) : 0) & 0xffu;
    }
    __device__ __forceinline__ uint32_t again(uint32_t w) const {
        uint32_t r = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) r |= code(byte_of(w, e) * before) << (8 * e);
        return r;
    }
};

// New rows [lo, hi) of a page, `front` earlier ones in front of them; x points
// at the row that becomes the page's row 0 (which may lie before the tensor).  The
// page (times heads, plus head) is looked at behind the rows' loads, so that its own
// load runs beside them; negative, there is none.
template <int D, int kType, bool kCodes>
__device__ void write_keys(const void *x, int64_t row_stride, const float *in_scale, int first_token, const uint16_t *mean,
                           int8_t *codes, float *scale, int64_t at, int front, int lo, int hi, uint32_t *part) {
    constexpr int kItems = kPage * D / 8 / kThreads;  // pieces of 8 channels of a row
    float v[kItems][8];
    uint32_t amax = 0;
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
        const int row = (it * kThreads + threadIdx.x) / (D / 8), c = threadIdx.x % (D / 8);
        if (row < lo || row >= hi) continue;
        if constexpr (kCodes) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(static_cast<const int8_t *>(x) + row * row_stride + 8 * c);
            const float s = in_scale[(first_token + row) / kPage];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[it][e] = byte_of(w[e >> 2], e & 3) * s;
        } else {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(x) + row * row_stride + 8 * c);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[it][e] = element<kType>(w[e >> 1], e & 1);
        }
        if (mean) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(mean + 8 * c);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[it][e] -= element<0>(w[e >> 1], e & 1);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = max(amax, magnitude(v[it][e]));
    }
    if (at < 0) return;
    codes += at * kPage * D, scale += at;
    const float scale_before = *scale;
    const Quantizer q(group_max(amax, part), scale_before, front > 0);
    if (threadIdx.x == 0) *scale = q.scale;
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
        const int row = (it * kThreads + threadIdx.x) / (D / 8), c = threadIdx.x % (D / 8);
        auto *dst = reinterpret_cast<u32x2 *>(codes + row * D + 8 * c);
        u32x2 w;
        if (row >= lo && row < hi) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
                w[e] = q.code(v[it][4 * e]) | q.code(v[it][4 * e + 1]) << 8 | q.code(v[it][4 * e + 2]) << 16 |
                       q.code(v[it][4 * e + 3]) << 24;
        } else if (q.grown && row < front) {
            w = *dst;
#pragma unroll
            for (int e = 0; e < 2; ++e) w[e] = q.again(w[e]);
        } else {
            continue;
        }
        *dst = w;
    }
}

// A page of V^T in LDS on its way between rows of tokens (a thread has 4 of them) and
// rows of channels: 68 bytes a channel, which spreads a wave's dwords over the banks.
constexpr int kTurn = kPage / 4 + 1;  // dwords of a channel
template <int D>
struct Turn {
    uint32_t at[D * kTurn];
    __device__ __forceinline__ uint32_t &dword(int channel, int quad) { return at[channel * kTurn + quad]; }
    // The thread's pieces of 16 bytes of a page's codes, contiguous over the workgroup.
    __device__ __forceinline__ void out(int8_t *codes) {
#pragma unroll
        for (int it = 0; it < kPage * D / 16 / kThreads; ++it) {
            const int i = it * kThreads + threadIdx.x;
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = dword(i / 4, 4 * (i % 4) + e);
            reinterpret_cast<u32x4 *>(codes)[i] = w;
        }
    }
    __device__ __forceinline__ void in(const int8_t *codes) {
#pragma unroll
        for (int it = 0; it < kPage * D / 16 / kThreads; ++it) {
            const int i = it * kThreads + threadIdx.x;
            const u32x4 w = reinterpret_cast<const u32x4 *>(codes)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) dword(i / 4, 4 * (i % 4) + e) = w[e];
        }
    }
};

template <int D, int kType>
__device__ void write_values(const void *x, int64_t row_stride, int8_t *codes, float *scale, int64_t at, int front, int lo,
                             int hi, uint32_t *part, Turn<D> &turn) {
    constexpr int kCh = D / 16;  // channels of a thread, times 4 tokens
    const int c = threadIdx.x % 16, t0 = 4 * (threadIdx.x / 16);
    typedef uint32_t Row __attribute__((ext_vector_type(kCh / 2)));
    float v[4][kCh];
    uint32_t amax = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int row = t0 + t;
        const bool fresh = row >= lo && row < hi;
        Row w = {};
        if (fresh) {
            w = *reinterpret_cast<const Row *>(static_cast<const uint16_t *>(x) + row * row_stride + kCh * c);
        }
#pragma unroll
        for (int e = 0; e < kCh; ++e) {
            v[t][e] = element<kType>(w[e >> 1], e & 1);
            amax = max(amax, magnitude(v[t][e]));
        }
    }
    if (at < 0) return;
    codes += at * kPage * D, scale += at;
    const float scale_before = *scale;
    const Quantizer q(group_max(amax, part), scale_before, front > 0);
    if (threadIdx.x == 0) *scale = q.scale;
    if (lo == 0 && hi == kPage) {  // a page of new tokens alone
#pragma unroll
        for (int e = 0; e < kCh; ++e)
            turn.dword(kCh * c + e, t0 / 4) = q.code(v[0][e]) | q.code(v[1][e]) << 8 | q.code(v[2][e]) << 16 | q.code(v[3][e]) << 24;
        __syncthreads();
        turn.out(codes);
        return;
    }
    uint32_t fresh = 0, earlier = 0;  // bytes of the thread's four tokens
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        fresh |= (t0 + t >= lo && t0 + t < hi ? 0xffu : 0u) << (8 * t);
        earlier |= (q.grown && t0 + t < front ? 0xffu : 0u) << (8 * t);
    }
    if (!(fresh | earlier)) return;
#pragma unroll
    for (int e = 0; e < kCh; ++e) {
        auto *dst = reinterpret_cast<uint32_t *>(codes + (kCh * c + e) * kPage + t0);
        uint32_t w = q.code(v[0][e]) | q.code(v[1][e]) << 8 | q.code(v[2][e]) << 16 | q.code(v[3][e]) << 24;
        if (fresh != 0xffffffffu) {
            const uint32_t old = *dst;
            const uint32_t kept = earlier ? (q.again(old) & earlier) | (old & ~earlier) : old;
            w = (w & fresh) | (kept & ~fresh);
        }
        *dst = w;
    }
}

// Workgroup (block of the sequence's new tokens * heads + head, 2 * sequence + (0: keys, 1: values)).
template <int D, int kType, bool kCodes>
__global__ __launch_bounds__(kThreads) void cache_append_kernel(
    const void *__restrict__ k, const float *__restrict__ k_in_scale, const void *__restrict__ v, int32_t len, int64_t k_sb,
    int64_t k_sh, int64_t k_sl, int64_t v_sb, int64_t v_sh, int64_t v_sl, const uint16_t *__restrict__ k_mean, Pages pages,
    const int32_t *__restrict__ new_lengths, int8_t *__restrict__ k_codes, int8_t *__restrict__ v_codes,
    float *__restrict__ k_scale, float *__restrict__ v_scale, int32_t *__restrict__ lengths_out) {
    __shared__ uint32_t part[kThreads / 64];
    __shared__ Turn<D> turn;
    const uint32_t h = blockIdx.x % pages.hkv, b = blockIdx.y >> 1, nth = blockIdx.x / pages.hkv;
    const bool keys = (blockIdx.y & 1) == 0;
    const int before = held(pages, b);
    const int fresh = min(new_lengths ? min(max(new_lengths[b], 0), len) : len, pages.width * kPage - before);
    if (blockIdx.x == 0 && keys && threadIdx.x == 0) lengths_out[b] = before + fresh;
    const int block = before / kPage + static_cast<int>(nth), base = block * kPage;
    const int lo = max(before - base, 0), hi = min(before + fresh - base, kPage);
    if (lo >= hi) return;
    const int page = page_of(pages, b, block);
    const int64_t at = page < 0 ? -1 : static_cast<int64_t>(page) * pages.hkv + h;
    const int first = base - before;  // token of the call that is the page's row 0 (negative: one held before)
    if (keys) {
        const int64_t off = b * k_sb + h * k_sh + first * k_sl;
        const void *x = kCodes ? static_cast<const void *>(static_cast<const int8_t *>(k) + off)
                               : static_cast<const void *>(static_cast<const uint16_t *>(k) + off);
        const float *in = kCodes ? k_in_scale + static_cast<int64_t>(b * pages.hkv + h) * ((len + kPage - 1) / kPage) : nullptr;
        write_keys<D, kType, kCodes>(x, k_sl, in, first, k_mean ? k_mean + static_cast<int64_t>(b * pages.hkv + h) * D : nullptr,
                                     k_codes, k_scale, at, lo, lo, hi, part);
    } else {
        write_values<D, kType>(static_cast<const uint16_t *>(v) + b * v_sb + h * v_sh + first * v_sl, v_sl,
                               v_codes, v_scale, at, lo, lo, hi, part, turn);
    }
}

template <int kType>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (kType == 0) return pack_bf16x2(a, b);
    else return pack_f16x2(a, b);
}

// Workgroup (block that the tokens read lie in * heads + head, 2 * sequence + (0:
// keys, 1: values)): rows of the output whose tokens lie in the block; zeros at and
// past the sequence's end and where the table names no page.
template <int D, int kType>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(
    const int8_t *__restrict__ k_codes, const int8_t *__restrict__ v_codes, const float *__restrict__ k_scale,
    const float *__restrict__ v_scale, Pages pages, const int32_t *__restrict__ starts, int32_t len,
    const uint16_t *__restrict__ k_mean, uint16_t *__restrict__ k, int64_t k_sb, int64_t k_sh, int64_t k_sl,
    uint16_t *__restrict__ v, int64_t v_sb, int64_t v_sh, int64_t v_sl) {
    __shared__ Turn<D> turn;
    const uint32_t h = blockIdx.x % pages.hkv, b = blockIdx.y >> 1, nth = blockIdx.x / pages.hkv;
    const bool keys = (blockIdx.y & 1) == 0;
    const int end = held(pages, b);
    const int start = starts ? min(max(starts[b], 0), pages.width * kPage) : 0;
    const int block = start / kPage + static_cast<int>(nth);
    const int64_t base = static_cast<int64_t>(block) * kPage;
    const int lo = static_cast<int>(max(start - base, static_cast<int64_t>(0)));
    const int hi = static_cast<int>(min(start + static_cast<int64_t>(len) - base, static_cast<int64_t>(kPage)));
    if (lo >= hi) return;
    const int page = base < end ? page_of(pages, b, block) : -1;
    const int seen = page < 0 ? 0 : static_cast<int>(min(end - base, static_cast<int64_t>(kPage)));  // rows that hold a token
    const int64_t at = static_cast<int64_t>(max(page, 0)) * pages.hkv + h;
    const int64_t first = base - start;  // output row of the block's row 0
    if (keys) {
        const int8_t *codes = k_codes + at * kPage * D;
        const float s = seen > 0 ? k_scale[at] : 0.0f;
        const uint16_t *mean = k_mean ? k_mean + static_cast<int64_t>(b * pages.hkv + h) * D : nullptr;
        uint16_t *out = k + b * k_sb + h * k_sh + first * k_sl;
#pragma unroll
        for (int it = 0; it < kPage * D / 8 / kThreads; ++it) {
            const int row = (it * kThreads + threadIdx.x) / (D / 8), c = threadIdx.x % (D / 8);
            if (row < lo || row >= hi) continue;
            u32x4 r = {};
            if (row < seen) {
                const u32x2 w = *reinterpret_cast<const u32x2 *>(codes + row * D + 8 * c);
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = byte_of(w[e >> 2], e & 3) * s;
                if (mean) {
                    const u32x4 m = *reinterpret_cast<const u32x4 *>(mean + 8 * c);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] += element<0>(m[e >> 1], e & 1);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = pack2<kType>(x[2 * e], x[2 * e + 1]);
            }
            *reinterpret_cast<u32x4 *>(out + row * k_sl + 8 * c) = r;
        }
    } else {
        constexpr int kCh = D / 16;  // channels of a thread, times 4 tokens
        const int c = threadIdx.x % 16, t0 = 4 * (threadIdx.x / 16);
        const int8_t *codes = v_codes + at * kPage * D;
        const float s = seen > 0 ? v_scale[at] : 0.0f;
        if (seen > 0) turn.in(codes);
        __syncthreads();
        uint16_t *out = v + b * v_sb + h * v_sh + first * v_sl;
        uint32_t w[kCh] = {};
        if (t0 < seen) {
#pragma unroll
            for (int e = 0; e < kCh; ++e) w[e] = turn.dword(kCh * c + e, t0 / 4);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int row = t0 + t;
            if (row < lo || row >= hi) continue;
            typedef uint32_t Row __attribute__((ext_vector_type(kCh / 2)));
            Row r = {};
            if (row < seen) {
#pragma unroll
                for (int e = 0; e < kCh / 2; ++e) r[e] = pack2<kType>(byte_of(w[2 * e], t) * s, byte_of(w[2 * e + 1], t) * s);
            }
            *reinterpret_cast<Row *>(out + row * v_sl + kCh * c) = r;
        }
    }
}

// What both calls ask of the cache, the table and the tensors.
int32_t check_cache(const char *what, int64_t batch, int64_t hkv, int64_t len, int64_t dim, int64_t width, int64_t pages,
                    const void *const *pointers, int n, const int64_t *strides, int multiple_k) {
    TU_REQUIRE(dim == 64 || dim == 128, "%s requires head_dim 64 or 128, got %lld", what, static_cast<long long>(dim));
    TU_REQUIRE(batch > 0 && hkv > 0 && len > 0 && batch <= 32767 && hkv <= 65535 && len <= 0x7fffff00,
               "%s sizes out of range", what);
    TU_REQUIRE(width > 0 && width <= 0x7fffffff / kPage - 1 && pages > 0 && pages <= 0x7fffffff,
               "%s block table or page count out of range", what);
    for (int i = 0; i < n; ++i) TU_REQUIRE(pointers[i], "%s pointers must be non-null", what);
    for (int i = 0; i < 4; ++i)
        TU_REQUIRE((reinterpret_cast<uintptr_t>(pointers[i]) & 15) == 0, "%s K/V and codes must be 16-byte aligned", what);
    for (int i = 0; i < 6; ++i)
        TU_REQUIRE(strides[i] % (i < 3 ? multiple_k : 8) == 0, "%s K/V rows must be 16-byte aligned", what);
    return 0;
}

}  // namespace
}  // namespace tu

extern "C" int32_t tu_kv_cache_append(const void *k, const float *k_in_scale, const void *v, int32_t dtype, int64_t batch,
                                      int64_t hkv, int64_t len, int64_t dim, int64_t k_sb, int64_t k_sh, int64_t k_sl,
                                      int64_t v_sb, int64_t v_sh, int64_t v_sl, const void *k_mean_bf16,
                                      const int32_t *block_table, int64_t width, const int32_t *lengths,
                                      const int32_t *new_lengths, int8_t *k_codes, int8_t *v_codes, float *k_scale,
                                      float *v_scale, int64_t pages, int32_t *lengths_out, void *stream) {
    using namespace tu;
    const void *pointers[] = {k, v, k_codes, v_codes, block_table, lengths, k_scale, v_scale, lengths_out};
    const int64_t strides[] = {k_sb, k_sh, k_sl, v_sb, v_sh, v_sl};
    if (check_cache("cache append", batch, hkv, len, dim, width, pages, pointers, 9, strides, k_in_scale ? 16 : 8)) return -1;
    TU_REQUIRE(dtype == 0 || dtype == 1, "cache append dtype must be 0 (bf16) or 1 (fp16), got %d", dtype);
    TU_REQUIRE((reinterpret_cast<uintptr_t>(k_mean_bf16) & 15) == 0, "cache append K mean must be 16-byte aligned");
    TU_REQUIRE(lengths_out != lengths, "cache append: the new lengths need memory of their own");
    // len tokens touch one page more where they do not start at a page's start
    const int64_t blocks = std::min<int64_t>((len + 2 * kPage - 2) / kPage, width);
    TU_REQUIRE(blocks * hkv <= kMostWgs, "cache append grid too large");
    if (require_gfx950()) return -1;
    const Pages p{block_table, lengths, static_cast<int32_t>(width), static_cast<int32_t>(pages), static_cast<uint32_t>(hkv)};
    const dim3 grid(static_cast<unsigned>(blocks * hkv), static_cast<unsigned>(2 * batch));
    hipStream_t s = static_cast<hipStream_t>(stream);
#define TU_APPEND(D, TYPE, CODES)                                                                                      \
    cache_append_kernel<D, TYPE, CODES><<<grid, kThreads, 0, s>>>(                                                     \
        k, k_in_scale, v, static_cast<int32_t>(len), k_sb, k_sh, k_sl, v_sb, v_sh, v_sl,                               \
        static_cast<const uint16_t *>(k_mean_bf16), p, new_lengths, k_codes, v_codes, k_scale, v_scale, lengths_out)
#define TU_APPEND_TYPES(D)                                                                                             \
    do {                                                                                                               \
        if (k_in_scale) {                                                                                              \
            if (dtype == 0) TU_APPEND(D, 0, true);                                                                     \
            else TU_APPEND(D, 1, true);                                                                                \
        } else if (dtype == 0) {                                                                                       \
            TU_APPEND(D, 0, false);                                                                                    \
        } else {                                                                                                       \
            TU_APPEND(D, 1, false);                                                                                    \
        }                                                                                                              \
    } while (0)
    if (dim == 128) TU_APPEND_TYPES(128);
    else TU_APPEND_TYPES(64);
#undef TU_APPEND_TYPES
#undef TU_APPEND
    return check_launch("tu_kv_cache_append");
}

extern "C" int32_t tu_kv_cache_read(const int8_t *k_codes, const int8_t *v_codes, const float *k_scale, const float *v_scale,
                                    int64_t pages, const int32_t *block_table, int64_t width, const int32_t *lengths,
                                    const int32_t *starts, const void *k_mean_bf16, void *k, void *v, int32_t dtype,
                                    int64_t batch, int64_t hkv, int64_t len, int64_t dim, int64_t k_sb, int64_t k_sh,
                                    int64_t k_sl, int64_t v_sb, int64_t v_sh, int64_t v_sl, void *stream) {
    using namespace tu;
    const void *pointers[] = {k, v, k_codes, v_codes, block_table, lengths, k_scale, v_scale};
    const int64_t strides[] = {k_sb, k_sh, k_sl, v_sb, v_sh, v_sl};
    if (check_cache("cache read", batch, hkv, len, dim, width, pages, pointers, 8, strides, 8)) return -1;
    TU_REQUIRE(dtype == 0 || dtype == 1, "cache read dtype must be 0 (bf16) or 1 (fp16), got %d", dtype);
    TU_REQUIRE((reinterpret_cast<uintptr_t>(k_mean_bf16) & 15) == 0, "cache read K mean must be 16-byte aligned");
    const int64_t blocks = starts ? (len + 2 * kPage - 2) / kPage : (len + kPage - 1) / kPage;
    TU_REQUIRE(blocks * hkv <= kMostWgs, "cache read grid too large");
    if (require_gfx950()) return -1;
    const Pages p{block_table, lengths, static_cast<int32_t>(width), static_cast<int32_t>(pages), static_cast<uint32_t>(hkv)};
    const dim3 grid(static_cast<unsigned>(blocks * hkv), static_cast<unsigned>(2 * batch));
    hipStream_t s = static_cast<hipStream_t>(stream);
#define TU_READ(D, TYPE)                                                                                               \
    cache_read_kernel<D, TYPE><<<grid, kThreads, 0, s>>>(                                                              \
        k_codes, v_codes, k_scale, v_scale, p, starts, static_cast<int32_t>(len),                                      \
        static_cast<const uint16_t *>(k_mean_bf16), static_cast<uint16_t *>(k), k_sb, k_sh, k_sl,                      \
        static_cast<uint16_t *>(v), v_sb, v_sh, v_sl)
    if (dim == 128) {
        if (dtype == 0) TU_READ(128, 0);
        else TU_READ(128, 1);
    } else if (dtype == 0) {
        TU_READ(64, 0);
    } else {
        TU_READ(64, 1);
    }
#undef TU_READ
    return check_launch("tu_kv_cache_read");
}
