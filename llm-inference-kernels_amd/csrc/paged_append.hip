// New tokens into a paged cache: the rotary embedding of q and k and the page
// writes of k and v, from the fused q|k|v projection's rows, in one launch.
//
// Row t of qkv is a token of sequence b (the one whose range of cu_tokens holds
// t; without cu_tokens row b is sequence b's newest token) at position
//   pos = seq_lens[b] - (cu_tokens[b + 1] - t)      (seq_lens[b] - 1),
// and for d < D/2 with the position's rows of the cos and sin tables
//   x'[d] = x[d] cos[d] - x[d + D/2] sin[d],
//   x'[d + D/2] = x[d + D/2] cos[d + D/2] + x[d] sin[d + D/2]
// in fp32, rounded once (the arithmetic of rope). The bytes bound it: each row
// is read and written once.
//
// A thread moves 8 dimensions and their partners D / 2 further of one head in
// 16-byte accesses; a workgroup's threads take one token's heads, so the table
// rows of a token are read through one CU's cache. The row's data is requested
// before the sequence, its length and the page are looked up, which is a chain
// of three loads. Measured: 9067 rows of 48 heads in bf16 42.2 us (5.3 TB/s, a large
// copy reaches 4.9); one row 1.9 us on the GPU, 5.0 with the call.
#include "paged_common.hpp"

namespace llmik {

namespace {

struct PagedAppendParams {
    const uint16_t* qkv;
    const void* cos;
    const void* sin;
    uint16_t* q_out;
    uint16_t* k;
    uint16_t* v;
    const int* table;
    const int* lens;
    const int* cu;
    long page_stride;
    int n_pages, max_pages, batch, n_heads, n_kv_heads, capacity, table_rows;
    FastDiv page;
};

template <bool BF>
__device__ __forceinline__ void halves_to_f32(const u32x4 raw, float (&v)[8]) {
    if constexpr (BF) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t x = raw[e];
            v[2 * e] = Half16<true>::to_f32((uint16_t)x);
            v[2 * e + 1] = Half16<true>::to_f32((uint16_t)(x >> 16));
        }
    } else {
        f16x8_to_f32(raw, v);
    }
}

// Eight table values as fp32, from the qkv type or fp32.
template <bool BF, bool F32>
__device__ __forceinline__ void table8(const void* t, long at, float (&v)[8]) {
    if constexpr (F32) {
        const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(t) + at);
        const f32x4 a = p[0], b = p[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = a[e];
            v[4 + e] = b[e];
        }
    } else {
        halves_to_f32<BF>(load16(static_cast<const uint16_t*>(t) + at), v);
    }
}

}  // namespace

// blockIdx.x: the row; blockIdx.y: its part of the heads. TPH threads per head.
template <bool BF, bool F32, int D>
__global__ __launch_bounds__(1024) void paged_append_kernel(PagedAppendParams p) {
    using Hf = Half16<BF>;
    constexpr int TPH = D / 16;
    const int t = blockIdx.x;
    const int idx = blockIdx.y * blockDim.x + threadIdx.x;
    const int lane = threadIdx.x & 63;
    const int heads = p.n_heads + 2 * p.n_kv_heads;
    const int head = idx / TPH, d = 8 * (idx % TPH);
    const bool work = head < heads;
    const uint16_t* src = p.qkv + ((long)t * heads + min(head, heads - 1)) * D + d;
    const u32x4 x1 = load16(src), x2 = load16(src + D / 2);

    // The row's sequence: as many as have their range's end at or before t.
    int b = t, ahead = 1;   // ahead: tokens of the sequence from this row on
    if (p.cu != nullptr) {
        b = 0;
        for (int i = 0; i < p.batch; i += 64) {   // every wave for itself
            const int end = i + lane < p.batch ? p.cu[i + lane + 1] : INT_MAX;
            b += __popcll(__ballot(end <= t));
        }
        if (b < p.batch) ahead = p.cu[b + 1] - t;
    }
    const int pos = b < p.batch ? max(p.lens[b], 0) - ahead : -1;   // (the lowest length: no overflow)
    const bool rotate = p.cos != nullptr;
    const bool live = pos >= 0 && pos < (rotate ? p.table_rows : INT_MAX);
    if (!work) return;

    const bool is_q = head < p.n_heads;
    u32x4 y1 = x1, y2 = x2;
    if (rotate && live && head < p.n_heads + p.n_kv_heads) {
        float c1[8], s1[8], c2[8], s2[8];
        const long row = (long)pos * D + d;
        table8<BF, F32>(p.cos, row, c1);
        table8<BF, F32>(p.sin, row, s1);
        table8<BF, F32>(p.cos, row + D / 2, c2);
        table8<BF, F32>(p.sin, row + D / 2, s2);
        float f1[8], f2[8];
        halves_to_f32<BF>(x1, f1);
        halves_to_f32<BF>(x2, f2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (BF) {
                float o1[2], o2[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int i = 2 * e + u;
                    o1[u] = fmaf(f1[i], c1[i], -(f2[i] * s1[i]));
                    o2[u] = fmaf(f2[i], c2[i], f1[i] * s2[i]);
                }
                y1[e] = Hf::pack(o1[0], o1[1]);
                y2[e] = Hf::pack(o2[0], o2[1]);
            } else {   // rope's rounding: with fp16 tables the same bits
                uint16_t l1, l2, h1, h2;
                rope_pair(f1[2 * e], f2[2 * e], c1[2 * e], s1[2 * e], c2[2 * e], s2[2 * e], l1, l2);
                rope_pair(f1[2 * e + 1], f2[2 * e + 1], c1[2 * e + 1], s1[2 * e + 1], c2[2 * e + 1], s2[2 * e + 1],
                          h1, h2);
                y1[e] = (uint32_t)l1 | ((uint32_t)h1 << 16);
                y2[e] = (uint32_t)l2 | ((uint32_t)h2 << 16);
            }
        }
    }
    uint16_t* dst;
    if (is_q) {
        if (!live) y1 = y2 = u32x4{0u, 0u, 0u, 0u};   // a row of no sequence
        dst = p.q_out + ((long)t * p.n_heads + head) * D + d;
    } else {
        if (!live || pos >= p.capacity) return;
        const uint32_t pi = p.page.div((uint32_t)pos);
        const int page = p.table[(long)b * p.max_pages + pi];
        if ((uint32_t)page >= (uint32_t)p.n_pages) return;   // unmapped
        const int kv = head - p.n_heads;
        const bool is_k = kv < p.n_kv_heads;
        const int slot = pos - (int)(pi * p.page.d);
        dst = (is_k ? p.k : p.v) + (long)page * p.page_stride +
              ((long)(is_k ? kv : kv - p.n_kv_heads) * p.page.d + slot) * D + d;
    }
    *reinterpret_cast<u32x4*>(dst) = y1;
    *reinterpret_cast<u32x4*>(dst + D / 2) = y2;
}

int launch_paged_append(const PagedAppend& a, hipStream_t stream) {
    PagedAppendParams p{};
    p.qkv = static_cast<const uint16_t*>(a.qkv);
    p.cos = a.cos;
    p.sin = a.sin;
    p.q_out = static_cast<uint16_t*>(a.q_out);
    p.k = static_cast<uint16_t*>(a.k);
    p.v = static_cast<uint16_t*>(a.v);
    p.table = a.table;
    p.lens = a.lens;
    p.cu = a.cu;
    p.page_stride = a.page_stride;
    p.n_pages = a.n_pages;
    p.max_pages = a.max_pages;
    p.batch = a.batch;
    p.n_heads = a.n_heads;
    p.n_kv_heads = a.n_kv_heads;
    p.capacity = (int)std::min((long)a.max_pages * a.page_size, kMaxPagedTokens);
    p.table_rows = a.table_rows;
    p.page = FastDiv::of((uint32_t)a.page_size);
    // One workgroup per row up to 512 threads, in whole waves.
    const int items = (a.n_heads + 2 * a.n_kv_heads) * (a.head_dim / 16);
    const int parts = (items + 511) / 512;
    const int threads = ((items + parts - 1) / parts + 63) / 64 * 64;
    const dim3 grid((unsigned)a.rows, (unsigned)((items + threads - 1) / threads));
    auto go = [&](auto bf, auto f32) {
        constexpr bool BF = decltype(bf)::value, F32 = decltype(f32)::value;
        if (a.head_dim == 128) paged_append_kernel<BF, F32, 128><<<grid, threads, 0, stream>>>(p);
        else paged_append_kernel<BF, F32, 64><<<grid, threads, 0, stream>>>(p);
    };
    using std::false_type;
    using std::true_type;
    if (a.bf16) a.table_f32 ? go(true_type{}, true_type{}) : go(true_type{}, false_type{});
    else a.table_f32 ? go(false_type{}, true_type{}) : go(false_type{}, false_type{});
    return check_launch();
}

}  // namespace llmik
