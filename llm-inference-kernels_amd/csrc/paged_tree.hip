// Attention of drafted token trees over a paged cache (paged_flash.hpp's tree form): the
// n drafted tokens of a sequence are its last n slots; each sees all cached tokens and,
// of the drafted ones, those whose bits its mask has (its ancestors and itself).
//
// All drafted tokens and query heads that read a KV head's keys share one pass over
// them, 128 rows at a time, so the cache's bytes bound it while they are few. The key
// tiles of the batch are cut into parts of about one length (Cutter): a row
// tile's parts are joined by a second kernel.
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

namespace {
constexpr int kJoinBatch = 8;   // parts that a thread requests at a time
constexpr int join_rows(int head_dim) { return 256 * 4 / head_dim; }   // of a workgroup: a thread has four channels
}  // namespace

template <bool BF, int D>
__global__ __launch_bounds__(256) void paged_tree_join_kernel(PagedFlashParams p) {
    using Hf = Half16<BF>;
    const int kvh = (int)(blockIdx.x % (uint32_t)p.c.n_kv_heads), cut = (int)(blockIdx.x / (uint32_t)p.c.n_kv_heads);
    if (cut >= p.records[0].count) return;
    const CutRecord t = p.records[cut];
    const int row = join_rows(D) * (int)blockIdx.y + (int)threadIdx.x / (D / 4);   // of the tile
    const int r = t.tile * kPfRows + row;
    if (r >= t.rows * (int)p.gqa.d || t.parts == 0) return;
    const int c4 = 4 * ((int)threadIdx.x % (D / 4));
    float top = kNoMax, sum = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int u0 = 0; u0 < t.parts; u0 += kJoinBatch) {
        f32x2 ml[kJoinBatch];
        f32x4 v[kJoinBatch];
#pragma unroll
        for (int u = 0; u < kJoinBatch; ++u) {
            const long at = part_row(p, t.slot + (uint32_t)(min(u0 + u, t.parts - 1) * t.fixed), kvh, row);
            ml[u] = *reinterpret_cast<const f32x2*>(p.part_ml + 2 * at);
            v[u] = *reinterpret_cast<const f32x4*>(p.part_o + at * D + c4);
        }
        float m = top;
#pragma unroll
        for (int u = 0; u < kJoinBatch; ++u) m = fmaxf(m, ml[u][0]);
        const float a = join_weight(top - m);
        top = m;
        sum *= a;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= a;
#pragma unroll
        for (int u = 0; u < kJoinBatch; ++u) {
            const bool in = u0 + u < t.parts;
            const float w = join_weight(ml[u][0] - m);
            sum = in ? fmaf(ml[u][1], w, sum) : sum;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = in ? fmaf(v[u][e], w, o[e]) : o[e];
        }
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;   // a row without keys is zero
    const int qi = (int)p.gqa.div((uint32_t)r);
    const long q_row = ((long)t.row0 + qi) * p.n_heads + kvh * (int)p.gqa.d + (r - qi * (int)p.gqa.d);
    *reinterpret_cast<u32x2*>(p.out + q_row * D + c4) =
        u32x2{Hf::pack(o[0] * inv, o[1] * inv), Hf::pack(o[2] * inv, o[3] * inv)};
}

// ---------------------------------------------------------------- host

namespace {

// The key tiles are cut for two workgroups per CU, into single tiles where there are few. us, a draft of 8 over 700
// tokens with 1, 2, 4 tiles or more 12.3, 13.1, 14.0; 30 drafts of 4 .. 24 over 200 .. 8000 tokens for 256, 384, 512,
// 768 workgroups 88.6, 70.2, 62.0, 76.3; one of 64 over 8192 28.8, 29.6, 30.4, 38.1.
constexpr int kTreePerCu = 2, kTreeLeast = 1;

struct PagedTreePlan {
    long row_tiles;      // of the call at most
    int target;
    uint32_t slots;      // 0: nothing is cut
    size_t off_o, off_records, bytes;
};

PagedTreePlan plan_tree(int batch, int rows, int n_heads, int n_kv_heads, int head_dim, long capacity, int cus) {
    PagedTreePlan pl{};
    const long all = (long)rows * (n_heads / n_kv_heads);
    pl.row_tiles = std::min((all + (long)batch * (kPfRows - 1)) / kPfRows, all / kPfRows + std::min(batch, rows));
    pl.target = std::max(kTreePerCu * cus / n_kv_heads, 1);
    if (capacity > (long)kTreeLeast * kPfTile) {
        // A row tile that is cut has more than one length's tiles: less than twice the target's parts.
        pl.slots = 2u * (uint32_t)pl.target;
        const size_t parts = (size_t)pl.slots * n_kv_heads * kPfRows;
        pl.off_o = align_up(parts * 2 * sizeof(float), 256);
        pl.off_records = pl.off_o + align_up(parts * head_dim * sizeof(float), 256);
        pl.bytes = pl.off_records + pl.slots / 2 * sizeof(CutRecord);
    }
    return pl;
}

template <bool BF, int D>
void launch_tree(const PagedFlashParams& p, long items, long cut_tiles, hipStream_t stream) {
    const unsigned grid = (unsigned)(items * p.c.n_kv_heads);
    if (p.s.cap_x != 0.0f) paged_tree_kernel<BF, D, true><<<grid, kPfThreads, 0, stream>>>(p);
    else paged_tree_kernel<BF, D, false><<<grid, kPfThreads, 0, stream>>>(p);
    if (p.slots == 0) return;
    const dim3 join((unsigned)(cut_tiles * p.c.n_kv_heads), (unsigned)(kPfRows / join_rows(D)));
    paged_tree_join_kernel<BF, D><<<join, 256, 0, stream>>>(p);
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
    }
    p.splits = 1;
    p.observe = INT_MAX;
    p.mask = mask;
    p.words = words;
    p.positions = positions;
    p.target = pl.target;
    p.least = pl.slots > 0 ? kTreeLeast : kUncut;
    p.slots = pl.slots;
    const long items = pl.row_tiles + (pl.slots > 0 ? pl.target : 0);
    const long cut = std::min(pl.row_tiles, (long)pl.target);   // (a tile that is cut has two parts at least)
    if (a.bf16)
        a.head_dim == 128 ? launch_tree<true, 128>(p, items, cut, stream)
                          : launch_tree<true, 64>(p, items, cut, stream);
    else
        a.head_dim == 128 ? launch_tree<false, 128>(p, items, cut, stream)
                          : launch_tree<false, 64>(p, items, cut, stream);
    return check_launch();
}

}  // namespace llmik
