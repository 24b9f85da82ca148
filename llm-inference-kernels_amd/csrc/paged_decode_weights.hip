// A decode step that records each token's attention weight: paged_decode.hpp's
// attention stores its scores (fp32, 4 bytes per query head and key beside the keys'
// 4 D per KV head) and each head's maximum and sum, and a second launch adds
//   weights[row(b), kvh, t] += sum over the KV head's G query heads of 2^(s - m) / l
// Every weight has one writer, so the sums do not depend on timing.
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

constexpr int kRecordThreads = 256, kRecordTokens = 1024;   // of a workgroup's turn

struct RecordParams {
    const float* scores;
    const float* row_ml;
    const int* lens;
    WeightsView w;
    int batch, n_heads, n_kv_heads, gqa, capacity, window, score_tokens;
};

}  // namespace

// The turns (a sequence's KV head and 1024 of its tokens) are numbered over the whole
// batch and taken by the workgroups in turn: the host does not know the lengths.
__global__ __launch_bounds__(kRecordThreads) void paged_record_kernel(RecordParams p) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int per = (p.batch + 63) / 64;
    const int b0 = min(lane * per, p.batch), b1 = min(b0 + per, p.batch);
    // A sequence's recorded keys [begin, end) and its turns for one KV head.
    auto keys_of = [&](int b, int& begin, int& end) {
        const int len = max(p.lens[b], 0);
        end = min(min(len, p.capacity), p.score_tokens);
        begin = min(max(len - p.window, 0), end);
        end = min(end, p.w.max_len);
        return end > begin ? (uint32_t)(end - begin + kRecordTokens - 1) / kRecordTokens : 0u;
    };
    uint32_t mine = 0;
    int begin, end;
    for (int b = b0; b < b1; ++b) mine += keys_of(b, begin, end) * (uint32_t)p.n_kv_heads;
    const uint32_t incl = wave_scan(mine), total = lane_u32(incl, 63);
    for (uint32_t x = blockIdx.x; x < total; x += gridDim.x) {
        const int at_lane = __ffsll((unsigned long long)__ballot(incl > x)) - 1;
        uint32_t first = lane_u32(incl - mine, at_lane), turns = 0;
        int b = at_lane * per;
        for (;; ++b) {   // ends: the lane's sequences hold turn x
            turns = keys_of(b, begin, end);
            if (x - first < turns * (uint32_t)p.n_kv_heads) break;
            first += turns * (uint32_t)p.n_kv_heads;
        }
        const int kvh = (int)((x - first) / turns);
        const int t0 = begin + kRecordTokens * (int)((x - first) - (uint32_t)kvh * turns);
        float* const w = weights_of(p.w, b, kvh);
        if (w == nullptr) continue;
        const long row = (long)b * p.n_heads + kvh * p.gqa;
        constexpr int kEach = kRecordTokens / kRecordThreads;
        float sum[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) sum[e] = 0.0f;
        for (int g = 0; g < p.gqa; ++g) {
            const float m = p.row_ml[2 * (row + g)], inv = p.row_ml[2 * (row + g) + 1];
            const float* s = p.scores + (row + g) * p.score_tokens;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int t = t0 + e * kRecordThreads + tid;
                const float x = t < end ? s[t] : -INFINITY;   // (-inf: no key)
                if (x > -INFINITY || x != x) sum[e] = fmaf(__builtin_amdgcn_exp2f(x - m), inv, sum[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int t = t0 + e * kRecordThreads + tid;
            if (t < end) w[t] += sum[e];
        }
    }
}

// ---------------------------------------------------------------- host

namespace {

struct DecodeWeightsPlan {
    PagedDecodePlan decode;
    int score_tokens;
    size_t off_ml, off_scores, bytes;
};

DecodeWeightsPlan plan_decode_weights(int batch, int n_heads, int n_kv_heads, int head_dim, long capacity,
                                      int max_len, int cus) {
    DecodeWeightsPlan pl{};
    pl.decode = plan_paged_decode(batch, n_heads, n_kv_heads, head_dim, capacity, cus);
    pl.score_tokens = (int)align_up((size_t)std::min(capacity, (long)max_len), 64);
    pl.off_ml = align_up(pl.decode.bytes, 256);
    pl.off_scores = pl.off_ml + align_up((size_t)batch * n_heads * 2 * sizeof(float), 256);
    pl.bytes = pl.off_scores + (size_t)batch * n_heads * pl.score_tokens * sizeof(float);
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

size_t paged_decode_weights_workspace(int batch, int n_heads, int n_kv_heads, int head_dim, long capacity,
                                      int max_len) {
    return plan_decode_weights(batch, n_heads, n_kv_heads, head_dim, capacity, max_len, device_cu_count()).bytes;
}

int launch_paged_decode_weights(const PagedLaunch& a, const PagedWeights& w, hipStream_t stream) {
    const int cus = device_cu_count();
    const long capacity = std::min((long)a.max_pages * a.page_size, kMaxPagedTokens);
    const DecodeWeightsPlan pl =
        plan_decode_weights(a.batch, a.n_heads, a.n_kv_heads, a.head_dim, capacity, w.max_len, cus);
    if (a.workspace == nullptr || a.workspace_bytes < pl.bytes)
        return set_error(LLMIK_ERR_WORKSPACE, "workspace too small (llmik_paged_decode_weights_workspace_size)");
    if ((long)pl.decode.workgroups > kMaxCounters)
        return set_error(LLMIK_ERR_UNSUPPORTED, "too many compute units for the workspace's counters");
    PagedDecodeParams p = paged_decode_params(a, pl.decode);
    char* ws = static_cast<char*>(a.workspace);
    p.row_ml = reinterpret_cast<float*>(ws + pl.off_ml);
    p.scores = reinterpret_cast<float*>(ws + pl.off_scores);
    p.score_tokens = pl.score_tokens;
    const bool uniform = a.page_size % 32 == 0;
    if (a.bf16)
        a.head_dim == 128 ? launch_scores<true, 128>(p, pl.decode.workgroups, uniform, stream)
                          : launch_scores<true, 64>(p, pl.decode.workgroups, uniform, stream);
    else
        a.head_dim == 128 ? launch_scores<false, 128>(p, pl.decode.workgroups, uniform, stream)
                          : launch_scores<false, 64>(p, pl.decode.workgroups, uniform, stream);
    const int st = check_launch();
    if (st != LLMIK_OK) return st;
    RecordParams r{p.scores, p.row_ml, a.lens, weights_view(w, a.n_kv_heads), a.batch, a.n_heads, a.n_kv_heads,
                   p.gqa, p.c.capacity, p.s.window, pl.score_tokens};
    const long turns = (long)a.batch * a.n_kv_heads * ((pl.score_tokens + kRecordTokens - 1) / kRecordTokens);
    paged_record_kernel<<<(unsigned)std::min(turns, 8L * cus), kRecordThreads, 0, stream>>>(r);
    return check_launch();
}

}  // namespace llmik
