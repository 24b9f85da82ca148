// Attention of drafted token trees over a paged cache (paged_flash.hpp's tree form): the
// n drafted tokens of a sequence are its last n slots; each sees all cached tokens and,
// of the drafted ones, those whose bits its mask has (its ancestors and itself).
//
// All drafted tokens and query heads that read a KV head's keys share one pass over
// them, 128 rows at a time, so the cache's bytes bound it while they are few. The key
// tiles of the batch are cut into parts of about one length (Cutter): a row
// tile's parts are joined by a second kernel. A row's mask is one 64-bit word for a tile
// of 64 keys, shifted to the tile's beginning; tiles of cached tokens need none.
//
// Measured (us under the tracer, kernel and join): 8 drafted tokens over 700 8.5 + 3.6, 64 over 8192
// 26 + 5.2, 32 sequences of 4 .. 24 over 200 .. 8000 60 + 5.4, all with 32 heads over 8 KV heads of 128
// (a call among others 11.2, 28.8, 64). The last reads 235 MB at 3.9 TB/s (8 drafted tokens over each of
// 32 x 8000: 1.05 GB in 196 us, 5.4 TB/s); of the second launch and look-ups take 8 us, a workgroup's 8 or 9
// tiles follow one another (the second product of a probability's pair is 3.5 us of them), and 17 MB of
// parts are written and read (eight waves in two teams, each with half of a part's keys, gain 1 us there and
// lose 1 at 700 tokens); the first is launches and look-ups.
#include "paged_flash.hpp"

namespace llmik {

template <bool BF, int D, bool EXACT>
__global__ __launch_bounds__(kPfThreads, 2) void paged_tree_kernel(PagedFlashParams p) {
    constexpr int kTileBytes = FlashLds<D>::kTileBytes;
    __shared__ __attribute__((aligned(16))) uint8_t s_k0[kTileBytes], s_k1[kTileBytes];
    __shared__ __attribute__((aligned(16))) uint8_t s_v0[kTileBytes], s_v1[kTileBytes];
    __shared__ int s_lo[4], s_hi[4];
    __shared__ uint32_t s_bad;
    paged_flash<BF, D, Flash::kTree, EXACT>(p, blockIdx.x, gridDim.x, {s_k0, s_k1, s_v0, s_v1, s_lo, s_hi, &s_bad});
}

// The parts of the cut sequences' rows, joined. A workgroup has kJoinRows rows, a wave
// every fourth part of them (eight requested at a time), a lane four channels of
// kRows rows one after the other; the waves are joined through LDS.
template <bool BF, int D>
__global__ __launch_bounds__(256) void paged_tree_join_kernel(PagedFlashParams p) {
    using Hf = Half16<BF>;
    constexpr int kWaves = 4, kAtOnce = 64 / (D / 4), kTurns = kJoinRows / kAtOnce, kBatch = 8 / kTurns;
    __shared__ __attribute__((aligned(16))) float s_o[kWaves][kTurns][64 * 4];
    __shared__ float s_m[kWaves][kTurns][64], s_l[kWaves][kTurns][64];
    const int kvh = (int)(blockIdx.x % (uint32_t)p.c.n_kv_heads), group = (int)(blockIdx.x / (uint32_t)p.c.n_kv_heads);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // The group's sequence: the last record that begins at or before it.
    const int count = p.records[0].count;
    int at = -1;
    for (int i = 0; i < count; i += 64)
        at += __popcll(__ballot(i + lane < count && p.records[min(i + lane, count - 1)].group <= group));
    if (at < 0) return;
    at = __builtin_amdgcn_readfirstlane(at);
    const CutRecord t = p.records[at];
    const int n_rows = t.rows * (int)p.gqa.d, r0 = kJoinRows * (group - t.group);
    if (r0 >= n_rows) return;
    const int c4 = 4 * (lane % (D / 4));
    auto row_of = [&](int turn) { return min(r0 + turn * kAtOnce + lane / (D / 4), n_rows - 1); };
    auto part_at = [&](int turn, int part) {
        const int r = row_of(turn), tile = r / kPfRows;
        return part_row(p, t.slot + (uint32_t)(part * t.fixed + tile), kvh, r - tile * kPfRows);
    };
    float top[kTurns], sum[kTurns];
    f32x4 o[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
        top[k] = kNoMax;
        sum[k] = 0.0f;
        o[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // N parts, of which those that `counts` says, into one.
    auto join = [&](int k, auto n, auto counts, const float* m, const float* l, const f32x4* v) {
        constexpr int N = decltype(n)::value;
        float most = top[k];
#pragma unroll
        for (int u = 0; u < N; ++u) most = fmaxf(most, counts(u) ? m[u] : kNoMax);
        const float a = join_weight(top[k] - most);
        top[k] = most;
        sum[k] *= a;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][e] *= a;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const float w = join_weight(m[u] - most);
            sum[k] = counts(u) ? fmaf(l[u], w, sum[k]) : sum[k];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[k][e] = counts(u) ? fmaf(v[u][e], w, o[k][e]) : o[k][e];
        }
    };
    for (int u0 = wave; u0 < t.parts; u0 += kWaves * kBatch) {
        float m[kTurns][kBatch], l[kTurns][kBatch];
        f32x4 v[kTurns][kBatch];
#pragma unroll
        for (int k = 0; k < kTurns; ++k)
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                f32x2 ml = {kNoMax, 0.0f};
                v[k][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (u0 + kWaves * u < t.parts) {   // (of the wave)
                    const long from = part_at(k, u0 + kWaves * u);
                    ml = *reinterpret_cast<const f32x2*>(p.part_ml + 2 * from);
                    v[k][u] = *reinterpret_cast<const f32x4*>(p.part_o + from * D + c4);
                }
                m[k][u] = ml[0];
                l[k][u] = ml[1];
            }
#pragma unroll
        for (int k = 0; k < kTurns; ++k)
            join(k, std::integral_constant<int, kBatch>{}, [&](int u) { return u0 + kWaves * u < t.parts; }, m[k], l[k],
                 v[k]);
    }
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
        s_m[wave][k][lane] = top[k];
        s_l[wave][k][lane] = sum[k];
        *reinterpret_cast<f32x4*>(&s_o[wave][k][4 * lane]) = o[k];
    }
    __syncthreads();
    if (wave >= kTurns) return;   // wave k: the rows of turn k
    const int k0 = wave;
    float m[kWaves], l[kWaves];
    f32x4 v[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        m[w] = s_m[w][k0][lane];
        l[w] = s_l[w][k0][lane];
        v[w] = *reinterpret_cast<const f32x4*>(&s_o[w][k0][4 * lane]);
    }
    top[0] = kNoMax;
    sum[0] = 0.0f;
    o[0] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    join(0, std::integral_constant<int, kWaves>{}, [](int) { return true; }, m, l, v);
    const int r = r0 + k0 * kAtOnce + lane / (D / 4);
    if (r >= n_rows) return;
    const float inv = sum[0] > 0.0f || sum[0] != sum[0] ? 1.0f / sum[0] : 0.0f;   // a row without keys is zero
    const int qi = (int)p.gqa.div((uint32_t)r);
    const long q_row = ((long)t.row0 + qi) * p.n_heads + kvh * (int)p.gqa.d + (r - qi * (int)p.gqa.d);
    *reinterpret_cast<u32x2*>(p.out + q_row * D + c4) =
        u32x2{Hf::pack(o[0][0] * inv, o[0][1] * inv), Hf::pack(o[0][2] * inv, o[0][3] * inv)};
}

// ---------------------------------------------------------------- host

namespace {

// Key tiles are cut for two workgroups per CU, or, where there are row tiles for at most a quarter of the CUs, for one:
// the sums of every part are written and read again, but of many sequences the ends are ragged. us, a call among others,
// for 1, 2, 3 workgroups: one draft of 64 over 8192 tokens 31.4, 31.2, 31.0, over 16000 41.2, 46.4, 46.4, over 30000
// 65.6, 66.4, 66.4, of 32 over 30000 43.0, 49.5, 49.4, two of 64 over 8192 41.9, 45.9, 46.5; eight of 64 over 2000 (128 row
// tiles) 45.6, 48.8, 48.5, 16 of 32 over 4000 80.1, 80.1, 80.2, 30 of 4 .. 24 over 200 .. 8000 96.1, 65.8, 74.2. Into
// single tiles where there are few: 8 over 700 tokens with 1, 2, 4 tiles or more 12.3, 13.1, 14.0 (this and below
// replayed from a graph, with probabilities of one part).
constexpr int kTreeLeast = 1;
// A part's sums, 64 KiB, are written and read again, which takes 0.026 us of the card's time, a tile 1.3 us of its
// workgroup's (1.6 with probabilities of two parts, a tenth of the root): of N pairs of tiles in parts of t the sum
// of 1.3 t and 0.026 N / t is least at t^2 = N / 50, and a row tile whose keys are less than twice that is better whole
// (t^2 = N / 25). us without this rule, with N / 50, with N / 25: 32 drafts of 16 over 200 tokens 27.2, 18.1, 18.1, over
// 600 33.7, 33.7, 27.0, 8 of 16 over 600 19.7, 18.0, 19.4, 16 of 32 over 500 30.0, 29.9, 27.6.
constexpr float kTreePartCost = 25.0f;

struct PagedTreePlan {
    long row_tiles;      // of the call at most
    int target;
    uint32_t slots;      // 0: nothing is cut
    int records;         // sequences whose tiles are cut, at most
    long groups;         // of rows that are joined, at most
    size_t off_o, off_records, bytes;
};

PagedTreePlan plan_tree(int batch, int rows, int n_heads, int n_kv_heads, int head_dim, long capacity, int cus) {
    PagedTreePlan pl{};
    const long all = (long)rows * (n_heads / n_kv_heads);
    pl.row_tiles = std::min((all + (long)batch * (kPfRows - 1)) / kPfRows, all / kPfRows + std::min(batch, rows));
    const int per_cu = 4 * pl.row_tiles * n_kv_heads <= cus ? 1 : 2;
    pl.target = std::max(per_cu * cus / n_kv_heads, 1);
    pl.records = std::max(std::min({batch, rows, pl.target}), 1);   // (a tile that is cut has two parts at least)
    pl.groups = all / kJoinRows + pl.records;
    // (As many rows as no launch of the join holds fill the card uncut.)
    if (capacity > (long)kTreeLeast * kPfTile && pl.groups * n_kv_heads * 256 < 1L << 32) {
        // A row tile that is cut has more than one length's tiles: less than twice the target's parts.
        pl.slots = 2u * (uint32_t)pl.target;
        const size_t parts = (size_t)pl.slots * n_kv_heads * kPfRows;
        pl.off_o = align_up(parts * 2 * sizeof(float), 256);
        pl.off_records = pl.off_o + align_up(parts * head_dim * sizeof(float), 256);
        pl.bytes = pl.off_records + pl.records * sizeof(CutRecord);
    }
    return pl;
}

template <bool BF, int D>
void launch_tree(const PagedFlashParams& p, long items, long groups, hipStream_t stream) {
    const unsigned grid = (unsigned)(items * p.c.n_kv_heads);
    if (p.s.cap_x != 0.0f) paged_tree_kernel<BF, D, true><<<grid, kPfThreads, 0, stream>>>(p);
    else paged_tree_kernel<BF, D, false><<<grid, kPfThreads, 0, stream>>>(p);
    if (p.slots == 0) return;
    paged_tree_join_kernel<BF, D><<<(unsigned)(groups * p.c.n_kv_heads), 256, 0, stream>>>(p);
}

}  // namespace

size_t paged_tree_workspace(int batch, int rows, int n_heads, int n_kv_heads, int head_dim, long capacity) {
    const PagedTreePlan pl = plan_tree(batch, rows, n_heads, n_kv_heads, head_dim, capacity, device_cu_count());
    return pl.slots > 0 ? kCounterBytes + pl.bytes : 0;
}

int launch_paged_tree(const PagedLaunch& a, const uint64_t* mask, int words, const int* positions,
                      hipStream_t stream) {
    PagedFlashParams p = flash_params(a);
    const PagedTreePlan pl =
        plan_tree(a.batch, a.rows, a.n_heads, a.n_kv_heads, a.head_dim, p.c.capacity, device_cu_count());
    if (pl.slots > 0) {
        if (a.workspace == nullptr || a.workspace_bytes < kCounterBytes + pl.bytes)
            return set_error(LLMIK_ERR_WORKSPACE, "workspace too small (llmik_paged_tree_workspace_size)");
        char* ws = static_cast<char*>(a.workspace) + kCounterBytes;
        p.part_ml = reinterpret_cast<float*>(ws);
        p.part_o = reinterpret_cast<float*>(ws + pl.off_o);
        p.records = reinterpret_cast<CutRecord*>(ws + pl.off_records);
        p.n_records = pl.records;
    }
    p.splits = 1;
    p.observe = INT_MAX;
    p.mask = mask;
    p.words = words;
    p.positions = positions;
    p.target = pl.target;
    p.least = pl.slots > 0 ? kTreeLeast : kUncut;
    p.slots = pl.slots;
    p.part_cost = a.n_kv_heads / kTreePartCost;
    const long items = pl.row_tiles + (pl.slots > 0 ? pl.target : 0);
    if (a.bf16)
        a.head_dim == 128 ? launch_tree<true, 128>(p, items, pl.groups, stream)
                          : launch_tree<true, 64>(p, items, pl.groups, stream);
    else
        a.head_dim == 128 ? launch_tree<false, 128>(p, items, pl.groups, stream)
                          : launch_tree<false, 64>(p, items, pl.groups, stream);
    return check_launch();
}

}  // namespace llmik
