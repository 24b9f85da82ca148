// A decode step that records each token's attention weight: paged_decode.hpp's
// attention stores its scores (fp32, 4 bytes per query head and key beside the keys'
// 4 D per KV head) and each head's maximum and sum, and a second launch adds
//   weights[row(b), kvh, t] += sum over the KV head's G query heads of 2^(s - m) / l
// Every weight has one writer, so the sums do not depend on timing.
//
// Bound: the cache's bytes, and the scores' (G / D of the keys' and values') twice. us, a call
// among others, plain decode against this: 48 sequences of 1500 .. 8192 tokens, 8 KV heads, bf16
// 134, 170; 64 of 4096 164, 210; one of 900 9.2, 13.8, one of 30000 28.3, 34.2. Under the tracer the
// first of these is 133.4 against 160.4 and 9.5: the writes among the reads cost 27, whatever their
// order, place or part of a line, and the second launch the rest (64 of 4096 35 and 11.3, one of 900
// 1.4 and 3.9). Adding the weights in the first launch, by the last of a sequence's workgroups:
// 900 tokens 13.7, 2000 17.5 instead of 15.7, 4 x 4000 33.6 instead of 26.9.
#include "paged_decode.hpp"

namespace llmik {

template <bool BF, int D, bool UNI, bool EXACT>
__global__ __launch_bounds__(kPdThreads, kPdPerCu) void paged_decode_scores_kernel(PagedDecodeParams p) {
    constexpr int kFloats = DecodeLds<D>::kFloats;
    __shared__ __attribute__((aligned(16))) float s_o[kPdWaves * kFloats];
    __shared__ float s_m[kPdWaves][16], s_l[kPdWaves][16];
    __shared__ uint32_t s_last;
    paged_decode<BF, D, UNI, EXACT, true>(p, blockIdx.x, gridDim.x,
                                          {s_o, s_o + kFloats, s_o + 2 * kFloats, s_o + 3 * kFloats, s_m, s_l, &s_last});
}

namespace {

constexpr int kRecordThreads = 256, kRecordTokens = 1024;   // of a workgroup's turn: four for each thread

}  // namespace

// The turns (a sequence's KV head and 1024 of its tokens) are numbered over the whole
// batch and taken by the workgroups in turn: the host does not know the lengths.
// ALIGNED: the weights' rows are aligned to 16 bytes.
template <bool ALIGNED>
__global__ __launch_bounds__(kRecordThreads) void paged_record_kernel(PagedDecodeParams p, WeightsView w) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int per = (p.c.batch + 63) / 64;
    const int b0 = min(lane * per, p.c.batch), b1 = min(b0 + per, p.c.batch);
    // A sequence's recorded keys [begin, end) and its turns for one KV head, from a multiple of 32 on.
    auto turns_of = [&](int b, int& begin, int& end) {
        const Keys k = keys_of(p, p.c.lens[b]);
        begin = k.begin;
        end = min(min(k.end, p.score_tokens), w.max_len);
        return end > begin ? (uint32_t)(end - begin / 32 * 32 + kRecordTokens - 1) / kRecordTokens : 0u;
    };
    uint32_t mine = 0;
    int begin = 0, end = 0;   // (the lane's only sequence's, where per is 1)
    for (int b = b0; b < b1; ++b) mine += turns_of(b, begin, end) * (uint32_t)p.c.n_kv_heads;
    const uint32_t incl = wave_scan(mine), total = lane_u32(incl, 63);
    const int own_begin = begin, own_end = end;
    for (uint32_t x = blockIdx.x; x < total; x += gridDim.x) {
        const int at = __ffsll((unsigned long long)__ballot(incl > x)) - 1;
        uint32_t first = lane_u32(incl - mine, at), turns = lane_u32(mine, at) / (uint32_t)p.c.n_kv_heads;
        int b = at;
        if (per == 1) {
            begin = __builtin_amdgcn_readlane(own_begin, at);
            end = __builtin_amdgcn_readlane(own_end, at);
        } else {
            for (b = at * per;; ++b) {   // ends: the lane's sequences hold turn x
                turns = turns_of(b, begin, end);
                if (x - first < turns * (uint32_t)p.c.n_kv_heads) break;
                first += turns * (uint32_t)p.c.n_kv_heads;
            }
        }
        const int kvh = (int)((x - first) / turns);
        const int t = begin / 32 * 32 + kRecordTokens * (int)((x - first) - (uint32_t)kvh * turns) + 4 * tid;
        float* const to = weights_of(w, b, kvh);
        if (to == nullptr || t >= end) continue;
        const bool whole = t >= begin && t + 4 <= end;
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f}, old = sum;
        if (whole && ALIGNED) old = *reinterpret_cast<const f32x4*>(to + t);
        const float* const ml = p.row_ml + 2 * ((long)b * p.n_heads + kvh * p.gqa);
        const float* const s = p.scores + score_tile(p, b, kvh, t / 32 * 32) + t % 32;
        for (int g0 = 0; g0 < p.gqa; g0 += 4) {   // four heads' scores requested at a time
            f32x4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const f32x4*>(s + 32 * min(g0 + u, p.gqa - 1));
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (g0 + u >= p.gqa) break;
                const float m = ml[2 * (g0 + u)], inv = ml[2 * (g0 + u) + 1];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float score = v[u][e];   // (-inf: no key)
                    if (score > -INFINITY || score != score)
                        sum[e] = fmaf(__builtin_amdgcn_exp2f(score - m), inv, sum[e]);
                }
            }
        }
        if (whole && ALIGNED) {
            *reinterpret_cast<f32x4*>(to + t) = old + sum;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (t + e >= begin && t + e < end) to[t + e] += sum[e];
        }
    }
}

// ---------------------------------------------------------------- host

namespace {

struct ScoresPlan {
    int tokens;   // of a sequence
    size_t off_scores, bytes;
};

ScoresPlan plan_scores(int batch, int n_heads, long capacity, int max_len) {
    ScoresPlan pl{};
    pl.tokens = (int)align_up((size_t)std::min(capacity, (long)max_len), 64);
    pl.off_scores = align_up((size_t)batch * n_heads * 2 * sizeof(float), 256);
    pl.bytes = pl.off_scores + (size_t)batch * n_heads * pl.tokens * sizeof(float);
    return pl;
}

template <bool BF, int D>
void launch_scores(const PagedDecodeParams& p, int workgroups, bool uniform, hipStream_t stream) {
    auto go = [&](auto uni, auto exact) {
        paged_decode_scores_kernel<BF, D, decltype(uni)::value, decltype(exact)::value>
            <<<workgroups, kPdThreads, 0, stream>>>(p);
    };
    using std::false_type;
    using std::true_type;
    if (p.s.cap_x != 0.0f) uniform ? go(true_type{}, true_type{}) : go(false_type{}, true_type{});
    else uniform ? go(true_type{}, false_type{}) : go(false_type{}, false_type{});
}

}  // namespace

size_t paged_decode_weights_scratch(int batch, int n_heads, long capacity, int max_len) {
    return plan_scores(batch, n_heads, capacity, max_len).bytes;
}

int launch_paged_decode_weights(const PagedLaunch& a, const PagedWeights& w, void* scratch, size_t scratch_bytes,
                                hipStream_t stream) {
    const int cus = device_cu_count();
    const long capacity = std::min((long)a.max_pages * a.page_size, kMaxPagedTokens);
    const PagedDecodePlan pl = plan_paged_decode(a.batch, a.n_heads, a.n_kv_heads, a.head_dim, capacity, cus);
    const ScoresPlan sc = plan_scores(a.batch, a.n_heads, capacity, w.max_len);
    if (a.workspace == nullptr || a.workspace_bytes < pl.bytes)
        return set_error(LLMIK_ERR_WORKSPACE, "workspace too small (llmik_paged_workspace_size)");
    if (scratch == nullptr || scratch_bytes < sc.bytes)
        return set_error(LLMIK_ERR_WORKSPACE, "scratch too small (llmik_paged_decode_weights_scratch_size)");
    if ((long)pl.workgroups > kMaxCounters)
        return set_error(LLMIK_ERR_UNSUPPORTED, "too many compute units for the workspace's counters");
    PagedDecodeParams p = paged_decode_params(a, pl);
    p.row_ml = static_cast<float*>(scratch);
    p.scores = reinterpret_cast<float*>(static_cast<char*>(scratch) + sc.off_scores);
    p.score_tokens = sc.tokens;
    const bool uniform = a.page_size % 32 == 0;
    if (a.bf16)
        a.head_dim == 128 ? launch_scores<true, 128>(p, pl.workgroups, uniform, stream)
                          : launch_scores<true, 64>(p, pl.workgroups, uniform, stream);
    else
        a.head_dim == 128 ? launch_scores<false, 128>(p, pl.workgroups, uniform, stream)
                          : launch_scores<false, 64>(p, pl.workgroups, uniform, stream);
    const int st = check_launch();
    if (st != LLMIK_OK) return st;
    const long turns = (long)a.batch * a.n_kv_heads * (sc.tokens / kRecordTokens + 2);
    const unsigned grid = (unsigned)std::min(turns, 8L * cus);
    const WeightsView view = weights_view(w, a.n_kv_heads);
    if (w.max_len % 4 == 0 && reinterpret_cast<uintptr_t>(w.weights) % 16 == 0)
        paged_record_kernel<true><<<grid, kRecordThreads, 0, stream>>>(p, view);
    else
        paged_record_kernel<false><<<grid, kRecordThreads, 0, stream>>>(p, view);
    return check_launch();
}

}  // namespace llmik
