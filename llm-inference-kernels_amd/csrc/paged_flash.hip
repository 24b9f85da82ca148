// Attention of prompts over a paged cache (paged_flash.hpp): the join of the parts
// that a row tile's keys are cut into, and the launches.
#include "paged_flash.hpp"

namespace llmik {

template <bool BF, int D, bool EXACT>
__global__ __launch_bounds__(kPfThreads, 2) void paged_flash_kernel(PagedFlashParams p) {
    constexpr int kTileBytes = FlashLds<D>::kTileBytes;
    __shared__ __attribute__((aligned(16))) uint8_t s_k0[kTileBytes], s_k1[kTileBytes];
    __shared__ __attribute__((aligned(16))) uint8_t s_v0[kTileBytes], s_v1[kTileBytes];
    __shared__ int s_lo[4], s_hi[4];
    __shared__ uint32_t s_bad;
    paged_flash<BF, D, false, EXACT>(p, blockIdx.x, gridDim.x, {s_k0, s_k1, s_v0, s_v1, s_lo, s_hi, &s_bad});
}

// Rows of a workgroup of the join: a thread has four channels of one.
constexpr int join_rows(int head_dim) { return 256 * 4 / head_dim; }

// The parts of the row tiles joined. The time is a chain of loads, so every thread has
// one (us, 512 rows of a prompt over 16000 tokens with 32 rows a workgroup and 8: 57.6,
// 56.3; 8 x 8 rows over 8000: 41.1, 39.0).
template <bool BF, int D>
__global__ __launch_bounds__(256) void paged_flash_join_kernel(PagedFlashParams p) {
    using Hf = Half16<BF>;
    const int kvh = (int)blockIdx.x % p.c.n_kv_heads;
    const uint32_t item = blockIdx.x / (uint32_t)p.c.n_kv_heads;
    RowTile ft;
    if (!find_tile(p, item, ft)) return;
    const int parts = __builtin_amdgcn_readfirstlane(keys_of_tile(p, ft).parts);
    const int n_rows = ft.rows * (int)p.gqa.d;
    if (parts == 1) return;
    static_assert(kPfRows % join_rows(D) == 0, "a workgroup's rows belong to one tile");
    const int c4 = 4 * ((int)threadIdx.x % (D / 4));
    const long at0 = ((long)item * p.c.n_kv_heads + kvh) * p.splits * kPfRows;
    const int row = join_rows(D) * (int)blockIdx.y + (int)threadIdx.x / (D / 4);   // of the tile
    const int r = ft.tile * kPfRows + row;
    if (r >= n_rows) return;
    float m[kMaxParts], l[kMaxParts], top = kNoMax;
    f32x4 v[kMaxParts];
#pragma unroll
    for (int u = 0; u < kMaxParts; ++u) {
        const long at = at0 + (long)min(u, parts - 1) * kPfRows + row;
        m[u] = p.part_ml[2 * at];
        l[u] = p.part_ml[2 * at + 1];
        v[u] = *reinterpret_cast<const f32x4*>(p.part_o + at * D + c4);
    }
#pragma unroll
    for (int u = 0; u < kMaxParts; ++u) top = fmaxf(top, m[u]);
    float sum = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < kMaxParts; ++u) {
        const float w = join_weight(m[u] - top);
        sum = u < parts ? fmaf(l[u], w, sum) : sum;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = u < parts ? fmaf(v[u][e], w, o[e]) : o[e];
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    const int qi = (int)p.gqa.div((uint32_t)r);
    const long q_row = ((long)ft.row0 + qi) * p.n_heads + kvh * (int)p.gqa.d + (r - qi * (int)p.gqa.d);
    *reinterpret_cast<u32x2*>(p.out + q_row * D + c4) =
        u32x2{Hf::pack(o[0] * inv, o[1] * inv), Hf::pack(o[2] * inv, o[3] * inv)};
}

// ---------------------------------------------------------------- host

namespace {

template <bool BF, int D>
void launch_flash_kernel(const PagedFlashParams& p, unsigned grid, hipStream_t stream) {
    if (p.s.cap_x != 0.0f) paged_flash_kernel<BF, D, true><<<grid, kPfThreads, 0, stream>>>(p);
    else paged_flash_kernel<BF, D, false><<<grid, kPfThreads, 0, stream>>>(p);
}

void launch_flash(const PagedLaunch& a, const PagedFlashParams& p, long workgroups, hipStream_t stream) {
    const unsigned grid = (unsigned)workgroups;
    if (a.bf16)
        a.head_dim == 128 ? launch_flash_kernel<true, 128>(p, grid, stream)
                          : launch_flash_kernel<true, 64>(p, grid, stream);
    else
        a.head_dim == 128 ? launch_flash_kernel<false, 128>(p, grid, stream)
                          : launch_flash_kernel<false, 64>(p, grid, stream);
}

}  // namespace

// Row tiles of a ragged call at most, and the parts that their keys are cut into where
// there are fewer than two workgroups per CU: at most as many as fill those.
struct PagedPrefillPlan {
    long tiles, base;
    int splits;
    size_t off_o, bytes;
};

namespace {
PagedPrefillPlan plan_prefill(int batch, int rows, int n_heads, int n_kv_heads, int head_dim, long capacity, int cus) {
    PagedPrefillPlan pl{};
    const long all = (long)rows * (n_heads / n_kv_heads);
    pl.tiles = std::min((all + (long)batch * (kPfRows - 1)) / kPfRows, all / kPfRows + std::min(batch, rows));
    pl.base = std::max(pl.tiles * n_kv_heads, 1L);
    // As for the longest sequence that the table holds; the join's launch must pay too.
    const long longest = std::min((capacity + kPfTile - 1) / kPfTile, 1L << 20);
    const long most = 2L * cus / pl.base;
    const long n = most > 1 ? std::min(most, (long)parts_of((uint32_t)longest, (uint32_t)pl.base)) : 1;
    pl.splits = n > 1 && 1300 * longest * (n - 1) / n > 3000 + 26 * pl.base * n ? (int)n : 1;
    if (pl.splits > 1) {
        const size_t parts = (size_t)pl.base * pl.splits * kPfRows;
        pl.off_o = align_up(parts * 2 * sizeof(float), 256);
        pl.bytes = pl.off_o + align_up(parts * head_dim * sizeof(float), 256);
    }
    return pl;
}
}  // namespace

size_t paged_prefill_workspace(int batch, int rows, int n_heads, int n_kv_heads, int head_dim, long capacity) {
    const PagedPrefillPlan pl =
        plan_prefill(batch, rows, n_heads, n_kv_heads, head_dim, capacity, device_cu_count());
    return pl.splits > 1 ? kCounterBytes + pl.bytes : 0;
}

int launch_paged_prefill(const PagedLaunch& a, hipStream_t stream) {
    PagedFlashParams p = flash_params(a);
    const PagedPrefillPlan pl =
        plan_prefill(a.batch, a.rows, a.n_heads, a.n_kv_heads, a.head_dim, p.c.capacity, device_cu_count());
    p.splits = pl.splits;
    p.base = (int)std::min(pl.base, (long)INT_MAX);
    if (pl.splits > 1) {
        if (a.workspace == nullptr || a.workspace_bytes < kCounterBytes + pl.bytes)
            return set_error(LLMIK_ERR_WORKSPACE, "workspace too small (llmik_paged_prefill_workspace_size)");
        char* ws = static_cast<char*>(a.workspace) + kCounterBytes;
        p.part_ml = reinterpret_cast<float*>(ws);
        p.part_o = reinterpret_cast<float*>(ws + pl.off_o);
    }
    launch_flash(a, p, pl.tiles * a.n_kv_heads * pl.splits, stream);
    if (pl.splits > 1) {
        const dim3 grid((unsigned)(pl.tiles * a.n_kv_heads), (unsigned)(kPfRows / join_rows(a.head_dim)));
        if (a.bf16)
            a.head_dim == 128 ? paged_flash_join_kernel<true, 128><<<grid, 256, 0, stream>>>(p)
                              : paged_flash_join_kernel<true, 64><<<grid, 256, 0, stream>>>(p);
        else
            a.head_dim == 128 ? paged_flash_join_kernel<false, 128><<<grid, 256, 0, stream>>>(p)
                              : paged_flash_join_kernel<false, 64><<<grid, 256, 0, stream>>>(p);
    }
    return check_launch();
}

}  // namespace llmik
