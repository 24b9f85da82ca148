// A cache that is bounded by attention weight: which tokens of a sequence stay, and
// the moves that bring kept (or accepted) tokens together.
//
// Selection. Of a sequence's n tokens the first f and the last r stay, and of those
// between them the `need` of the largest weight, ties to the lowest slot. The weights,
// as integers of the same order, are searched by digits from the top: a histogram of
// the 8 bits below what is settled gives the digit of the need-th largest, until all that share
// its digits stay (four times at most).
// Then every wave counts, in a segment of its own, the weights above that value and
// those equal to it, and after a sum over the waves writes its slots in order.
// Bound: a chain of reads and barriers, the waves wait 62 % of the time (8192 tokens of 8 KV
// heads 9.5 us, 64 x 8 x 3500 .. 6000 14.4; with one histogram and the weights read anew for
// every digit 26, 29). Where a sequence has more candidates than LDS holds they are read again for every
// digit and count, by one workgroup: of 8 KV heads 36000 tokens 26 us, 40000 48, 100000 110, 32 x 40000 87,
// 16 x 100000 220.
//
// Compaction. Token kept[i] goes to slot start + i. No entry lies before its new slot
// (kept[i] >= start + i; others are not moved), so a workgroup that takes the entries
// in order, loads a chunk of them, waits, and then stores it, never overwrites what a
// later chunk reads: the moves are in place, whatever the order of the entries. What
// runs side by side are the sequences, KV heads, K and V, and slices of the rows'
// channels. Bound: the bytes that move, twice (16 sequences' 2048 of 2300 .. 6000 tokens, 268 MB:
// 66 us, 4.1 TB/s); a drafted tree's few tokens: the launch.
#include "paged_common.hpp"

namespace llmik {

namespace {

// ---------------------------------------------------------------- selection

constexpr int kSelWaves = 16;   // of a workgroup at most
constexpr int kSelCached = 36864;   // of 160 KiB of LDS, 16 for the rest
// Copies of the histogram, a lane's by its number: the weights' exponents are few, and additions to one place
// wait for each other. (Their bins lie in different banks.)
constexpr int kSelCopies = 8, kSelCopy = 256 + 4;

struct SelectParams {
    WeightsView w;
    const int* lens;
    int* kept;       // [batch, n_kv_heads, keep]
    int* new_lens;   // [batch]
    int keep, first, recent;
    int cached;      // candidates that LDS holds
};

// A weight as an integer of the same order: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) { return lane_u32(wave_scan(v), 63); }

}  // namespace

struct SelectLds {
    uint32_t hist[kSelCopies * kSelCopy];
    uint32_t count[256];
    uint32_t above[kSelWaves], equal[kSelWaves];
    uint32_t digit, rest, all;   // all: the value's digits so far leave no more than stay
};

// The candidates' `need` largest, of n: their slots, in order, to `out`. CACHED: in LDS,
// read once; else every pass reads them again.
template <bool CACHED, int THREADS>
__device__ __forceinline__ void select_largest(const float* w, int n, int need, int first, int* out, uint32_t* s_value,
                                               SelectLds& s) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t none = order_of(0.0f);   // where the sequence has no row
    auto read = [&](int i) { return w != nullptr ? order_of(w[i]) : none; };
    auto value = [&](int i) {
        if constexpr (CACHED) return s_value[i];
        else return read(i);
    };
    for (int i = tid; i < kSelCopies * kSelCopy; i += THREADS) s.hist[i] = 0u;
    __syncthreads();
    uint32_t* const hist = s.hist + (lane & (kSelCopies - 1)) * kSelCopy;
    if constexpr (CACHED) {   // with the first digit's histogram
        for (int i0 = 0; i0 < n; i0 += 4 * THREADS) {
            uint32_t x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = read(min(i0 + u * THREADS + tid, n - 1));
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i0 + u * THREADS + tid < n) {
                    s_value[i0 + u * THREADS + tid] = x[u];
                    atomicAdd(&hist[x[u] >> 24], 1u);
                }
        }
    }

    // ---- the need-th largest value ----
    uint32_t found = 0, rest = (uint32_t)need;   // of the top digits; its rank among those with these
    int shift = 24;
#pragma unroll 1
    for (;; shift -= 8) {   // until all with these digits stay
        for (int i0 = 0; i0 < n && !(CACHED && shift == 24); i0 += 4 * THREADS) {
            uint32_t x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = value(min(i0 + u * THREADS + tid, n - 1));
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i0 + u * THREADS + tid < n && (shift == 24 || x[u] >> (shift + 8) == found))
                    atomicAdd(&hist[x[u] >> shift & 255u], 1u);
        }
        __syncthreads();
        if (tid < 256) {
            uint32_t all = 0;
#pragma unroll
            for (int c = 0; c < kSelCopies; ++c) {
                all += s.hist[c * kSelCopy + tid];
                s.hist[c * kSelCopy + tid] = 0u;
            }
            s.count[tid] = all;
        }
        __syncthreads();
        if (wave == 0) {   // lane l: digits 255 - 4 l .. 252 - 4 l, from the top
            uint32_t c[4], mine = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) mine += c[e] = s.count[255 - 4 * lane - e];
            const uint32_t upto = wave_scan(mine);
            const int at = __ffsll((unsigned long long)__ballot(upto >= rest)) - 1;   // (all are >= rest together)
            if (lane == at) {
                uint32_t r = rest - (upto - mine), digit = 255u - 4u * lane, here = c[0];
                bool more = true;
#pragma unroll
                for (int e = 0; e < 3; ++e) {
                    more = more && r > c[e];
                    r -= more ? c[e] : 0u;
                    digit -= more ? 1u : 0u;
                    here = more ? c[e + 1] : here;
                }
                s.digit = digit;
                s.rest = r;
                s.all = r == here ? 1u : 0u;
            }
        }
        __syncthreads();
        found = found << 8 | s.digit;
        rest = s.rest;
        if (shift == 0 || s.all != 0) break;
    }
    // ---- every wave's segment: what lies above the value, and what equals it (the first `rest` stay) ----
    constexpr int kWaves = THREADS / kWave;
    const int seg = ((n + kWaves - 1) / kWaves + 63) / 64 * 64;
    const int i_begin = min(wave * seg, n), i_end = min((wave + 1) * seg, n);
    uint32_t above = 0, equal = 0;
    for (int i0 = i_begin; i0 < i_end; i0 += 256) {
        uint32_t x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = value(min(i0 + 64 * u + lane, n - 1));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool in = i0 + 64 * u + lane < i_end;
            above += in && x[u] >> shift > found;
            equal += in && x[u] >> shift == found;
        }
    }
    above = wave_sum(above);
    equal = wave_sum(equal);
    if (lane == 0) {
        s.above[wave] = above;
        s.equal[wave] = equal;
    }
    __syncthreads();
    // The sums of the waves before: a lane has one's.
    const uint32_t a_lane = lane < wave ? s.above[lane & (kSelWaves - 1)] : 0u;
    const uint32_t e_lane = lane < wave ? s.equal[lane & (kSelWaves - 1)] : 0u;
    uint32_t at_above = wave_sum(a_lane), at_equal = wave_sum(e_lane);
    auto before = [](uint64_t m) {   // of the lanes in front of this one
        return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
    };
    for (int i0 = i_begin; i0 < i_end; i0 += 256) {
        uint32_t x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = value(min(i0 + 64 * u + lane, n - 1));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + 64 * u + lane;
            const bool is_equal = i < i_end && x[u] >> shift == found;
            const uint64_t eq = __ballot(is_equal), ab = __ballot(i < i_end && x[u] >> shift > found);
            const uint32_t eq_before = at_equal + before(eq);
            if ((ab >> lane & 1u) || (is_equal && eq_before < rest))
                out[first + at_above + before(ab) + min(eq_before, rest)] = first + i;
            at_above += (uint32_t)__popcll(ab);
            at_equal += (uint32_t)__popcll(eq);
        }
    }
}

// One workgroup per (sequence, KV head).
template <int THREADS>
__global__ __launch_bounds__(THREADS) void paged_select_kernel(SelectParams p) {
    extern __shared__ uint32_t s_value[];
    __shared__ SelectLds s_all;
    const int tid = threadIdx.x;
    const int b = (int)blockIdx.x / p.w.n_kv_heads, kvh = (int)blockIdx.x - b * p.w.n_kv_heads;
    const int len = min(max(p.lens[b], 0), p.w.max_len);
    int* const out = p.kept + (long)blockIdx.x * p.keep;
    if (kvh == 0 && tid == 0) p.new_lens[b] = min(len, p.keep);
    if (len <= p.keep) {
        for (int i = tid; i < p.keep; i += THREADS) out[i] = i < len ? i : -1;
        return;
    }
    const float* const w = weights_of(p.w, b, kvh);
    const int n = len - p.first - p.recent;   // the candidates: > need, as first + recent <= keep < len
    const int need = p.keep - p.first - p.recent;
    for (int i = tid; i < p.first; i += THREADS) out[i] = i;
    for (int i = tid; i < p.recent; i += THREADS) out[p.first + need + i] = len - p.recent + i;
    if (need == 0) return;
    const float* const from = w != nullptr ? w + p.first : nullptr;
    if (n <= p.cached) select_largest<true, THREADS>(from, n, need, p.first, out, s_value, s_all);
    else select_largest<false, THREADS>(from, n, need, p.first, out, s_value, s_all);
}

int launch_paged_select(const PagedWeights& w, const int* lens, int batch, int n_kv_heads, int keep, int first,
                        int recent, int* kept, int* new_lens, hipStream_t stream) {
    const int cached = std::min(w.max_len, kSelCached);
    const SelectParams p{weights_view(w, n_kv_heads), lens, kept, new_lens, keep, first, recent, cached};
    // Waves and LDS go by the rows' width, which bounds the lengths; the lengths themselves are on the device. Eight
    // waves where they read a whole row in one turn of four weights a thread, else sixteen. us, 16, 8, 4 waves, sequences
    // of 8 KV heads x tokens in rows that end with them: 1 x 2000 6.6, 5.9, 7.4, 256 x 2000 31.1, 18.5, 16.4, 1 x 4000 7.1,
    // 7.8, 64 x 4000 10.7, 11.1, 64 x 3500 .. 6000 14.4, 13.6, 64 x 7000 15.7, 18.2, 1 x 8192 9.5, 11.5, 17.4. Short
    // sequences in wide rows pay for the width: 256 x 2000 in rows of 2000, 8192, 32768 17.7, 30.5, 46.8 (sixteen waves,
    // then one workgroup per CU), 64 x 3500 .. 6000 in rows of 6016, 20480 and more 14.3, 19.
    const unsigned grid = (unsigned)(batch * n_kv_heads);
    if (cached <= 4 * 512) paged_select_kernel<512><<<grid, 512, (size_t)cached * 4, stream>>>(p);
    else paged_select_kernel<1024><<<grid, 1024, (size_t)cached * 4, stream>>>(p);
    return check_launch();
}

// ---------------------------------------------------------------- compaction

namespace {

constexpr int kCompactBatch = 8;   // rows that a thread holds at a time

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

// Workgroup (b, kvh, part).
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

    if (part == 2 * p.slices) {   // the weights: moved by slots (no pages), those behind the kept ones become 0
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
        const int moves = min(count, stop - start);
        for (int i0 = 0; i0 < moves; i0 += threads) {
            const int i = i0 + tid, t = i < moves ? source(i) : -1;
            const float x = t >= 0 && t < p.w.max_len ? w[t] : 0.0f;
            __syncthreads();
            if (t >= 0) w[start + i] = x;
        }
        __syncthreads();
        for (int i = count + tid; i < stop - start; i += threads) w[start + i] = 0.0f;
        return;
    }

    const int chunks = D / 8 / p.slices;              // of a slice
    const int rows = threads / chunks;                // that the workgroup requests at a time
    const int slice = part % p.slices;
    uint16_t* const base = part < p.slices ? p.k : p.v;
    const int* const table_row = p.c.table + (long)b * p.c.max_pages;
    const int row = tid / chunks, d = 8 * (slice * chunks + tid % chunks);
    const long head_at = (long)kvh * p.c.page.d * D + d;
    // Without branches, so that all of a thread's requests of one kind are on their way together: an
    // entry that moves nothing looks up and reads the first place that there is.
    for (int i0 = 0; i0 < p.n; i0 += rows * kCompactBatch) {
        int t[kCompactBatch], page[kCompactBatch], page2[kCompactBatch];
#pragma unroll
        for (int u = 0; u < kCompactBatch; ++u) t[u] = kept[min(i0 + u * rows + row, p.n - 1)];
#pragma unroll
        for (int u = 0; u < kCompactBatch; ++u) {
            const int i = i0 + u * rows + row;
            t[u] = i < p.n && t[u] < len && t[u] > start + i ? t[u] : -1;
            page[u] = table_row[p.c.page.div((uint32_t)max(t[u], 0))];
            page2[u] = table_row[t[u] < 0 ? 0u : p.c.page.div((uint32_t)(start + i))];
        }
        u32x4 x[kCompactBatch];
        long to[kCompactBatch];
#pragma unroll
        for (int u = 0; u < kCompactBatch; ++u) {
            const bool ok = t[u] >= 0 && (uint32_t)page[u] < (uint32_t)p.c.n_pages &&
                            (uint32_t)page2[u] < (uint32_t)p.c.n_pages;   // (neither unmapped)
            auto place = [&](int slot, int pg) {
                return (long)pg * p.c.page_stride + head_at + (slot - (int)(p.c.page.div((uint32_t)slot) * p.c.page.d)) * D;
            };
            to[u] = ok ? place(start + i0 + u * rows + row, page2[u]) : -1L;
            x[u] = load16(base + (ok ? place(t[u], page[u]) : (long)d));
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the chunk is in registers before any of it is overwritten
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kCompactBatch; ++u)
            if (to[u] >= 0) *reinterpret_cast<u32x4*>(base + to[u]) = x[u];
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
    // Slices of 128 bytes, the L2's lines, or of 64 where there are few workgroups. us, 1, 4, 16 sequences of 8 KV
    // heads, 2048 .. 4096 kept tokens of heads of 128, 2 slices 23.0, 17.2, 66, 4 slices 16.8, 20.9, 80.
    const int pairs = a.batch * a.n_kv_heads;
    p.slices = a.head_dim / 64 * (pairs <= 16 ? 2 : 1);
    p.parts = 2 * p.slices + (p.w.w != nullptr ? 1 : 0);
    // Threads for four pieces each, up to 1024: us, with 64, 128, 256, 512, 1024 threads 24 entries 4.0, 4.3, 5.4, 7.8,
    // 16.6 (32 sequences), 600 entries 13.9, 9.4, 6.7, 5.2, 6.3, 4096 entries 85, 49, 27, 19, 17 (one).
    const long pieces = (long)n * (a.head_dim / 8 / p.slices);
    const int threads = (int)std::min(std::max((pieces / 4 + 63) / 64 * 64, p.w.w != nullptr ? 256L : 64L), 1024L);
    const unsigned grid = (unsigned)(pairs * p.parts);
    if (a.head_dim == 128) paged_compact_kernel<128><<<grid, threads, 0, stream>>>(p);
    else paged_compact_kernel<64><<<grid, threads, 0, stream>>>(p);
    return check_launch();
}

}  // namespace llmik
