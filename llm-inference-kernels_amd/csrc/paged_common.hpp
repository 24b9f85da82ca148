// Shared by the kernels of the paged KV cache (paged_decode.hip, paged_flash.hip):
// the two 16-bit types, the cache's addressing and the score options.
//
// The cache is k, v [n_pages, n_kv_heads, page_size, D]; token t of sequence b
// lies in page page_table[b][t / page_size] at slot t % page_size. page_size is
// a multiple of 8, so eight consecutive tokens starting at a multiple of 8 (an
// octet) always lie in one page, one row behind the other: kernels look pages
// up once per octet. Entries outside [0, n_pages) are unmapped pages: no load
// goes there and their tokens are masked.
#pragma once

#include <algorithm>
#include <type_traits>
#include <climits>

#include "device_common.hpp"
#include "llmik_internal.hpp"

namespace llmik {

typedef __bf16 bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2eF = 1.4426950408889634f;

// fp16 or bf16 values as 16-bit words, with the products and the (round to
// nearest even) conversions of each.
template <bool BF>
struct Half16;
template <>
struct Half16<false> {
    static __device__ __forceinline__ float to_f32(uint16_t b) { return (float)__builtin_bit_cast(f16, b); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const f16x2 h = __builtin_convertvector(f32x2{a, b}, f16x2);
        return __builtin_bit_cast(uint32_t, h);
    }
    static __device__ __forceinline__ float add_pair(uint32_t p, float acc) {   // acc + both values
        const f16x2 one = {(f16)1.0f, (f16)1.0f};
        return __builtin_amdgcn_fdot2(as_f16x2(p), one, acc, false);
    }
    static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
};
template <>
struct Half16<true> {
    static __device__ __forceinline__ float to_f32(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const bf16x2 h = __builtin_convertvector(f32x2{a, b}, bf16x2);
        return __builtin_bit_cast(uint32_t, h);
    }
    static __device__ __forceinline__ float add_pair(uint32_t p, float acc) {
        const bf16x2 one = {(bf16)1.0f, (bf16)1.0f};
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p), one, acc, false);
    }
    static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
};

// Division of 0 <= n < 2^31 by a fixed divisor d >= 1: n / d = (n * mul) >> (32
// + shift) with shift = ceil(log2 d) - 1 and mul = floor(2^(32 + shift) / d) + 1
// <= 2^32 - 1 for d that is no power of two (n e < 2^(32 + shift) for the
// rounding error e = mul d - 2^(32 + shift) <= d <= 2^(shift + 1), as n < 2^31);
// a power of two is a shift (mul = 0).
struct FastDiv {
    uint32_t d, mul, shift;
    static FastDiv of(uint32_t d) {
        FastDiv f{d, 0, 0};
        while ((1ull << f.shift) < d) ++f.shift;
        if ((d & (d - 1)) != 0) {
            --f.shift;
            f.mul = (uint32_t)((1ull << (32 + f.shift)) / d + 1);
        }
        return f;
    }
    __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
        return mul ? (uint32_t)(((uint64_t)n * mul) >> 32) >> shift : n >> shift;
    }
};

// The cache as the kernels see it. Strides in elements of 16 bits.
struct PagedView {
    const uint16_t* k;
    const uint16_t* v;
    const int* table;     // [batch, max_pages]
    const int* lens;      // [batch]
    long page_stride;
    int n_pages, max_pages, batch, n_kv_heads, capacity;   // capacity: max_pages * page_size tokens
    FastDiv page;
};

// Element offset of the row of token t (an octet's first), KV head kvh, of the
// sequence with this table row; -1 where the token lies at or behind `end` or
// its page is unmapped. Without branches: every lane loads a table entry (the
// first one instead of those behind the end).
template <int D>
__device__ __forceinline__ long octet_offset(const PagedView& c, const int* table_row, int kvh, int t, int end) {
    const bool in = t < end;
    const uint32_t pi = in ? c.page.div((uint32_t)t) : 0u;
    const int page = table_row[pi];
    const int slot = t - (int)(pi * c.page.d);
    const long at = (long)page * c.page_stride + (long)kvh * (long)(c.page.d * D) + slot * D;
    return in && (uint32_t)page < (uint32_t)c.n_pages ? at : -1L;
}

// publish_load16's 8-byte form.
__device__ __forceinline__ u32x2 publish_load8(__amdgpu_buffer_rsrc_t r, uint32_t voff) {
    return __builtin_amdgcn_raw_buffer_load_b64(r, (int)voff, 0, kPublishAux);
}

// A running maximum starts here rather than at -inf: differences of two such are
// then numbers, and states without a key join like all others (their sums are 0).
constexpr float kNoMax = -1e30f;
// The least weight of sums that are joined: 0 would make NaN of an infinity in V, which reaches every row
// that sees it. (Of finite sums it adds less than fp32 keeps.)
constexpr float kMinWeight = 1.1754944e-38f;
__device__ __forceinline__ float join_weight(float d) { return fmaxf(__builtin_amdgcn_exp2f(d), kMinWeight); }
constexpr float kPShift = 8.0f;   // p is held as 2^8 p: fp16 keeps its full precision down to 2^-22

// Scores in the log2 domain. A cap: cap * tanh(s / cap) with tanh(x) = 1 - 2 /
// (e^2x + 1), as exp2 and one reciprocal. That is exact to about 2^-22 of the cap, up
// to a cap of kPlainCap 2^-16, less than the products' own rounding. Above it small scores
// would lose their bits (of 4096 2^-10), so there |x| < 1/2 goes by tanh's series (to
// x^15; the next term is below 2^-26 of the sum) and all scores are exact to 2^-21 of
// themselves.
constexpr float kPlainCap = 64.0f;
struct ScoreOpts {
    float scale_log2;   // softmax_scale * log2(e)
    float cap_in;       // 2 log2(e) * softmax_scale / softcap, or 0
    float cap_log2;     // softcap * log2(e)
    float cap_x;        // softmax_scale / softcap above kPlainCap, or 0
    const float* slopes;
    int window;         // keys per query, INT_MAX where unlimited
};
__device__ __forceinline__ float capped_part(float s, float cap_in) {   // (tanh(x) - 1) / 2
    return __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(s * cap_in));
}
__device__ __forceinline__ float capped(float s, float cap_in, float cap_log2) {
    return fmaf(2.0f * cap_log2, capped_part(s, cap_in), cap_log2);
}

__device__ __forceinline__ float tanh_series(float x) {   // |x| < 1/2
    const float y = x * x;
    float p = -929569.0f / 638512875.0f;
    p = fmaf(p, y, 21844.0f / 6081075.0f);
    p = fmaf(p, y, -1382.0f / 155925.0f);
    p = fmaf(p, y, 62.0f / 2835.0f);
    p = fmaf(p, y, -17.0f / 315.0f);
    p = fmaf(p, y, 2.0f / 15.0f);
    p = fmaf(p, y, -1.0f / 3.0f);
    return fmaf(p * y, x, x);
}
__device__ __forceinline__ float capped_tanh(float s, const ScoreOpts& o) {   // the score over the cap
    const float x = s * o.cap_x;
    return fabsf(x) < 0.5f ? tanh_series(x) : capped(s, o.cap_in, 1.0f);
}

// The kernels' views of a call.
inline PagedView paged_view(const PagedLaunch& a) {
    PagedView c{};
    c.k = static_cast<const uint16_t*>(a.k);
    c.v = static_cast<const uint16_t*>(a.v);
    c.table = a.table;
    c.lens = a.lens;
    c.page_stride = a.page_stride;
    c.n_pages = a.n_pages;
    c.max_pages = a.max_pages;
    c.batch = a.batch;
    c.n_kv_heads = a.n_kv_heads;
    c.capacity = (int)std::min((long)a.max_pages * a.page_size, kMaxPagedTokens);
    c.page = FastDiv::of((uint32_t)a.page_size);
    return c;
}
inline ScoreOpts score_opts(const PagedLaunch& a) {
    ScoreOpts s{};
    s.scale_log2 = a.softmax_scale * kLog2eF;
    if (a.softcap > 0.0f) {
        s.cap_in = 2.0f * kLog2eF * (a.softmax_scale / a.softcap);
        s.cap_log2 = a.softcap * kLog2eF;
        s.cap_x = a.softcap > kPlainCap ? a.softmax_scale / a.softcap : 0.0f;
    }
    s.slopes = a.slopes;
    s.window = a.window > 0 ? a.window : INT_MAX;
    return s;
}

// Each token's accumulated attention weight, as the kernels see it.
struct WeightsView {
    float* w;           // [n_rows, n_kv_heads, max_len], or null
    const int* rows;    // [batch], or null: row b is sequence b's
    int n_rows, max_len, n_kv_heads;
};

inline WeightsView weights_view(const PagedWeights& a, int n_kv_heads) {
    return {static_cast<float*>(a.weights), a.rows, a.n_rows, a.max_len, n_kv_heads};
}

// The weights of sequence b, KV head kvh; null where it has no row.
__device__ __forceinline__ float* weights_of(const WeightsView& v, int b, int kvh) {
    const int row = v.rows ? v.rows[b] : b;
    return v.w != nullptr && (uint32_t)row < (uint32_t)v.n_rows
               ? v.w + ((long)row * v.n_kv_heads + kvh) * v.max_len : nullptr;
}

// Those of two 16-bit values that are infinities or NaN; zeros in place of the others.
template <bool BF>
__device__ __forceinline__ uint32_t not_finite2(uint32_t x) {
    constexpr uint32_t inf = BF ? 0x7F80u : 0x7C00u;
    return ((x & inf) == inf ? x & 0xFFFFu : 0u) | ((x & (inf << 16)) == inf << 16 ? x & 0xFFFF0000u : 0u);
}

// max / sum over lanes l and l ^ 32, or l and l ^ 16.
__device__ __forceinline__ float xor32_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor32_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float xor16_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor16_sum(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);   // row_bcast 15, 31
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
    return v;
}
__device__ __forceinline__ uint32_t lane_u32(uint32_t v, int lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

}  // namespace llmik
