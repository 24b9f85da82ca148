// A cache that is bounded by attention weight: which tokens of a sequence stay, and
// the moves that bring kept (or accepted) tokens together.
//
// Selection. Of a sequence's n tokens the first f and the last r stay, and of those
// between them the `need` of the largest weight, ties to the lowest slot. The weights,
// as integers of the same order, are searched by digits from the top: a histogram of
// the 8 bits below what is settled gives the digit of the need-th largest, four times.
// Then every wave counts, in a segment of its own, the weights above that value and
// those equal to it, and after a sum over the waves writes its slots in order.
//
// Compaction. Token kept[i] goes to slot start + i. No entry lies before its new slot
// (kept[i] >= start + i; others are not moved), so a workgroup that takes the entries
// in order, loads a chunk of them, waits, and then stores it, never overwrites what a
// later chunk reads: the moves are in place, whatever the order of the entries. What
// runs side by side are the sequences, KV heads, K and V, and slices of the rows'
// channels.
#include "paged_common.hpp"

namespace llmik {

namespace {

// ---------------------------------------------------------------- selection

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / kWave;

struct SelectParams {
    WeightsView w;
    const int* lens;
    int* kept;       // [batch, n_kv_heads, keep]
    int* new_lens;   // [batch]
    int keep, first, recent;
};

// A weight as an integer of the same order: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) { return lane_u32(wave_scan(v), 63); }

}  // namespace

// One workgroup per (sequence, KV head).
__global__ __launch_bounds__(kSelThreads) void paged_select_kernel(SelectParams p) {
    __shared__ uint32_t s_hist[256];
    __shared__ uint32_t s_above[kSelWaves], s_equal[kSelWaves];
    __shared__ uint32_t s_digit, s_rest;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = (int)blockIdx.x / p.w.n_kv_heads, kvh = (int)blockIdx.x - b * p.w.n_kv_heads;
    const int len = min(max(p.lens[b], 0), p.w.max_len);
    int* const out = p.kept + (long)blockIdx.x * p.keep;
    if (kvh == 0 && tid == 0) p.new_lens[b] = min(len, p.keep);
    if (len <= p.keep) {
        for (int i = tid; i < p.keep; i += kSelThreads) out[i] = i < len ? i : -1;
        return;
    }
    const float* const w = weights_of(p.w, b, kvh);
    const int lo = p.first, hi = len - p.recent;   // the candidates; lo + recent <= keep < len
    const int need = p.keep - p.first - p.recent;
    for (int i = tid; i < p.first; i += kSelThreads) out[i] = i;
    for (int i = tid; i < p.recent; i += kSelThreads) out[p.first + need + i] = hi + i;
    if (need == 0) return;
    auto value = [&](int t) { return w != nullptr ? order_of(w[t]) : order_of(0.0f); };

    // ---- the need-th largest value ----
    uint32_t found = 0, rest = (uint32_t)need;   // of the top digits; its rank among those with these
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) s_hist[tid] = 0u;
        __syncthreads();
        for (int t0 = lo; t0 < hi; t0 += kSelThreads) {
            const int t = t0 + tid;
            const uint32_t x = t < hi ? value(t) : 0u;
            bool in = t < hi && (shift == 24 || x >> (shift + 8) == found);
            const uint32_t d = x >> shift & 255u;
            if (shift == 24) {   // few different exponents: a lane adds for all of its digit
                uint64_t left = __ballot(in);
                while (left != 0) {
                    const int l = __ffsll((unsigned long long)left) - 1;
                    const uint64_t same = __ballot(in && d == lane_u32(d, l));
                    if (lane == l) atomicAdd(&s_hist[d], (uint32_t)__popcll(same));
                    left &= ~same;
                }
            } else if (in) {
                atomicAdd(&s_hist[d], 1u);
            }
        }
        __syncthreads();
        if (wave == 0) {   // lane l: digits 255 - 4 l .. 252 - 4 l, from the top
            uint32_t n[4], mine = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) mine += n[e] = s_hist[255 - 4 * lane - e];
            const uint32_t upto = wave_scan(mine);
            const int at = __ffsll((unsigned long long)__ballot(upto >= rest)) - 1;   // (all are >= rest together)
            if (lane == at) {
                uint32_t r = rest - (upto - mine);
                int e = 0;
                while (e < 3 && r > n[e]) r -= n[e++];
                s_digit = 255u - 4u * lane - e;
                s_rest = r;
            }
        }
        __syncthreads();
        found = found << 8 | s_digit;
        rest = s_rest;
    }
    // ---- every wave's segment: what lies above the value, and what equals it (the first `rest` stay) ----
    const int n = hi - lo;
    const int seg = ((n + kSelWaves - 1) / kSelWaves + 63) / 64 * 64;
    const int t_begin = lo + min(wave * seg, n), t_end = lo + min((wave + 1) * seg, n);
    uint32_t above = 0, equal = 0;
    for (int t = t_begin + lane; t < t_end; t += 64) {
        const uint32_t x = value(t);
        above += x > found;
        equal += x == found;
    }
    above = wave_sum(above);
    equal = wave_sum(equal);
    if (lane == 0) {
        s_above[wave] = above;
        s_equal[wave] = equal;
    }
    __syncthreads();
    uint32_t at_above = 0, at_equal = 0;
    for (int i = 0; i < wave; ++i) {
        at_above += s_above[i];
        at_equal += s_equal[i];
    }
    const uint64_t below = (1ull << lane) - 1;
    for (int t0 = t_begin; t0 < t_end; t0 += 64) {
        const int t = t0 + lane;
        const uint32_t x = t < t_end ? value(t) : 0u;
        const bool is_equal = t < t_end && x == found;
        const uint64_t eq = __ballot(is_equal), ab = __ballot(t < t_end && x > found);
        const uint32_t eq_before = at_equal + (uint32_t)__popcll(eq & below);
        const bool stays = (ab >> lane & 1u) || (is_equal && eq_before < rest);
        if (stays)
            out[p.first + at_above + (uint32_t)__popcll(ab & below) + min(eq_before, rest)] = t;
        at_above += (uint32_t)__popcll(ab);
        at_equal += (uint32_t)__popcll(eq);
    }
}

int launch_paged_select(const PagedWeights& w, const int* lens, int batch, int n_kv_heads, int keep, int first,
                        int recent, int* kept, int* new_lens, hipStream_t stream) {
    const SelectParams p{weights_view(w, n_kv_heads), lens, kept, new_lens, keep, first, recent};
    paged_select_kernel<<<(unsigned)(batch * n_kv_heads), kSelThreads, 0, stream>>>(p);
    return check_launch();
}

// ---------------------------------------------------------------- compaction

namespace {

constexpr int kCompactBatch = 4;   // rows that a thread holds at a time

struct CompactParams {
    PagedView c;
    uint16_t* k;
    uint16_t* v;
    const int* kept;
    long kept_stride;       // of a sequence
    long kept_head_stride;  // 0: one list for all heads
    const int* starts;      // or null: 0
    WeightsView w;
    int n;
    int slices;             // of a row's channels
    int parts;              // workgroups of a (sequence, KV head): 2 slices, and one for the weights if there are any
};

}  // namespace

// Workgroup (b, kvh, part). LOG: log2 of the 16-byte chunks of a slice.
template <int D>
__global__ __launch_bounds__(1024) void paged_compact_kernel(CompactParams p) {
    __shared__ int s_count;
    const int tid = threadIdx.x, threads = blockDim.x;
    const int part = (int)blockIdx.x % p.parts, bh = (int)blockIdx.x / p.parts;
    const int b = bh / p.c.n_kv_heads, kvh = bh - b * p.c.n_kv_heads;
    const int* const kept = p.kept + b * p.kept_stride + kvh * p.kept_head_stride;
    const int start = p.starts ? p.starts[b] : 0;
    const int len = min(max(p.c.lens[b], 0), p.c.capacity);
    if (start < 0 || start >= len) return;
    // Entry i's source, or -1 where nothing is moved (slot start + i < capacity: the source is not before it).
    auto source = [&](int i) {
        const int t = i < p.n ? kept[i] : -1;
        return t < len && t > start + i ? t : -1;   // (start + i <= t: no overflow where it counts; n <= 2^30)
    };

    if (part == 2 * p.slices) {   // the weights: moved alike, those behind the kept ones become 0
        float* const w = weights_of(p.w, b, kvh);
        if (w == nullptr) return;
        const int stop = min(len, p.w.max_len);
        if (tid == 0) s_count = p.n;
        __syncthreads();
        for (int i = tid; i < p.n; i += threads)
            if (kept[i] < 0) {   // the first such ends the list
                atomicMin(&s_count, i);
                break;
            }
        __syncthreads();
        const int count = s_count;
        for (int i0 = 0; i0 < stop - start; i0 += threads) {
            const int i = i0 + tid, t = i < count ? source(i) : -1;
            const bool move = t >= 0 && start + i < stop;
            const bool clear = i >= count && i < stop - start;
            const float x = move && t < p.w.max_len ? w[t] : 0.0f;
            __syncthreads();
            if (move || clear) w[start + i] = x;
        }
        return;
    }

    const int chunks = D / 8 / p.slices;              // of a slice
    const int rows = threads / chunks;                // that the workgroup moves at a time
    const int slice = part % p.slices;
    uint16_t* const base = part < p.slices ? p.k : p.v;
    const int* const table_row = p.c.table + (long)b * p.c.max_pages;
    const int row = tid / chunks, d = 8 * (slice * chunks + tid % chunks);
    auto address = [&](int t) -> uint16_t* {   // null where the page is unmapped
        const uint32_t pi = p.c.page.div((uint32_t)t);
        const int page = table_row[pi];
        if ((uint32_t)page >= (uint32_t)p.c.n_pages) return nullptr;
        return base + (long)page * p.c.page_stride + ((long)kvh * p.c.page.d + (t - (int)(pi * p.c.page.d))) * D + d;
    };
    for (int i0 = 0; i0 < p.n; i0 += rows * kCompactBatch) {
        u32x4 x[kCompactBatch];
        uint16_t* to[kCompactBatch];
#pragma unroll
        for (int u = 0; u < kCompactBatch; ++u) {
            const int i = i0 + u * rows + row, t = source(i);
            to[u] = nullptr;
            if (t >= 0) {
                const uint16_t* from = address(t);
                if (from != nullptr) {
                    to[u] = address(start + i);
                    x[u] = load16(from);
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the chunk is in registers before any of it is overwritten
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kCompactBatch; ++u)
            if (to[u] != nullptr) *reinterpret_cast<u32x4*>(to[u]) = x[u];
    }
}

int launch_paged_compact(const PagedLaunch& a, const PagedWeights& w, const int* kept, int kept_heads, int n,
                         const int* starts, hipStream_t stream) {
    CompactParams p{};
    p.c = paged_view(a);
    p.k = const_cast<uint16_t*>(p.c.k);
    p.v = const_cast<uint16_t*>(p.c.v);
    p.kept = kept;
    p.kept_stride = (long)kept_heads * n;
    p.kept_head_stride = kept_heads > 1 ? n : 0;
    p.starts = starts;
    p.w = weights_view(w, a.n_kv_heads);
    p.n = n;
    p.slices = 1;
    p.parts = 2 * p.slices + (p.w.w != nullptr ? 1 : 0);
    const unsigned grid = (unsigned)(a.batch * a.n_kv_heads * p.parts);
    if (a.head_dim == 128) paged_compact_kernel<128><<<grid, 1024, 0, stream>>>(p);
    else paged_compact_kernel<64><<<grid, 1024, 0, stream>>>(p);
    return check_launch();
}

}  // namespace llmik
