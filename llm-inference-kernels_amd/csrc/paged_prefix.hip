// Decode attention of a batch whose sequences share their first tokens: one launch
// reads the shared prefix once for all rows (paged_flash.hpp, rows = the batch's
// queries of a KV head) and each sequence's own tokens (paged_decode.hpp), a second
// one joins a row's parts: those of the prefix, then its own.
//
// The two kinds of workgroups run beside each other: the prefix's are bound by their
// chain of products, exponentials and waits (one wave per SIMD: 46 % of its cycles wait,
// products take 4 us of 25), the others by memory. Measured, GPU us: 64 sequences behind
// 8192 tokens 30.1 (in launches of their own 37.1), of which the join is 4.9 (17 parts a
// row, written and read in fp32); 6 behind 1500 10.9 (16.0), two launches of dependent
// reads; 64 behind 4096 28, where decode attention, which reads the prefix 64 times,
// takes 110.
#include "paged_decode.hpp"
#include "paged_flash.hpp"

namespace llmik {

template <bool BF, int D, bool UNI, bool EXACT>
__global__ __launch_bounds__(kPfThreads, 2) void paged_prefix_kernel(PagedFlashParams f, PagedDecodeParams d,
                                                                     uint32_t flash_wgs) {
    static_assert(kPfThreads == kPdThreads, "one workgroup size for both");
    constexpr int kTileBytes = FlashLds<D>::kTileBytes;
    static_assert(kTileBytes >= DecodeLds<D>::kFloats * 4, "a wave's sums fit a tile's place");
    __shared__ __attribute__((aligned(16))) uint8_t s_k0[kTileBytes], s_k1[kTileBytes];
    __shared__ __attribute__((aligned(16))) uint8_t s_v0[kTileBytes], s_v1[kTileBytes];
    __shared__ int s_lo[4], s_hi[4];
    __shared__ uint32_t s_flag;
    __shared__ float s_m[kPdWaves][16], s_l[kPdWaves][16];
    if (blockIdx.x < flash_wgs)
        paged_flash<BF, D, Flash::kPrefix, EXACT>(f, blockIdx.x, flash_wgs, {s_k0, s_k1, s_v0, s_v1, s_lo, s_hi, &s_flag});
    else
        paged_decode<BF, D, UNI, EXACT>(d, blockIdx.x - flash_wgs, gridDim.x - flash_wgs,
                                 {reinterpret_cast<float*>(s_k0), reinterpret_cast<float*>(s_k1),
                                  reinterpret_cast<float*>(s_v0), reinterpret_cast<float*>(s_v1), s_m, s_l, &s_flag});
}

namespace {
constexpr int kJoinBatch = 10;   // parts that a lane requests at a time
}  // namespace

// The lanes' two halves take every other one of a row's parts, a lane four channels:
// up to twenty parts in one round trip (all by one thread, eight at a time: 8.0 us
// instead of 5.0 for 64 sequences behind 8192 tokens).
template <bool BF, int D>
__global__ __launch_bounds__(256) void paged_prefix_join_kernel(const float* part_o, const float* part_ml,
                                                                uint16_t* out, int parts, int rows, FastDiv per_kv,
                                                                FastDiv gqa) {
    using Hf = Half16<BF>;
    constexpr int kRows = 128 / D;   // of a wave
    const int lane = threadIdx.x & 63, half = lane >> 5;
    // Rows as the parts': [n_kv_heads, batch, gqa].
    const int row = (int)(blockIdx.x * 4 + (threadIdx.x >> 6)) * kRows + (lane & 31) / (D / 4);
    const int c4 = 4 * (lane % (D / 4));
    if (row >= rows) return;   // (both halves)
    const long at0 = (long)row * parts;
    float top = kNoMax, sum = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int u0 = half; u0 < parts; u0 += 2 * kJoinBatch) {
        f32x2 ml[kJoinBatch];
        f32x4 v[kJoinBatch];
#pragma unroll
        for (int u = 0; u < kJoinBatch; ++u) {
            const long at = at0 + min(u0 + 2 * u, parts - 1);
            ml[u] = *reinterpret_cast<const f32x2*>(part_ml + 2 * at);
            v[u] = *reinterpret_cast<const f32x4*>(part_o + at * D + c4);
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
            const bool in = u0 + 2 * u < parts;
            const float w = join_weight(ml[u][0] - m);
            sum = in ? fmaf(ml[u][1], w, sum) : sum;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = in ? fmaf(v[u][e], w, o[e]) : o[e];
        }
    }
    const float m = xor32_max(top), a = join_weight(top - m);
    sum = xor32_sum(sum * a);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = xor32_sum(o[e] * a);
    if (half != 0) return;
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;   // a row without keys is zero
    const uint32_t kvh = per_kv.div((uint32_t)row), r = (uint32_t)row - kvh * per_kv.d;
    const uint32_t b = gqa.div(r), head = kvh * gqa.d + (r - b * gqa.d);
    const uint32_t n_heads = (uint32_t)rows / per_kv.d * gqa.d;
    *reinterpret_cast<u32x2*>(out + ((long)b * n_heads + head) * D + c4) =
        u32x2{Hf::pack(o[0] * inv, o[1] * inv), Hf::pack(o[2] * inv, o[3] * inv)};
}

// ---------------------------------------------------------------- host

namespace {

struct PagedPrefixPlan {
    int row_tiles, splits, chunk;
    size_t off_o, off_ml, bytes;
};

// The prefix's parts lie behind the decode kernel's workspace.
PagedPrefixPlan plan_prefix(int batch, int n_heads, int n_kv_heads, int head_dim, long capacity, int prefix_len,
                            int cus) {
    PagedPrefixPlan pl{};
    const long rows = (long)batch * (n_heads / n_kv_heads);
    pl.row_tiles = (int)((rows + kPfRows - 1) / kPfRows);
    const long base = std::max((long)pl.row_tiles * n_kv_heads, 1L);
    // Splits of the prefix: two workgroups per CU, but beyond one per CU only in parts
    // of eight tiles, as every part's results are written and read again, and never in
    // less than two tiles. us, 64 sequences behind 8192 tokens, 16 and 32 splits 29.4,
    // 39.7; 2 sequences behind 4096, 16 and 32 splits 13.2, 12.4.
    const long tiles = ((long)prefix_len + kPfTile - 1) / kPfTile;
    const long splits =
        std::max(1L, std::min({2L * cus / base, std::max(cus / base, tiles / 8), (tiles + 1) / 2, 64L}));
    pl.chunk = (int)((tiles + splits - 1) / splits) * kPfTile;   // (prefix_len <= kMaxPagedTokens)
    pl.splits = (int)(((long)prefix_len + pl.chunk - 1) / pl.chunk);
    pl.off_ml = align_up(paged_decode_workspace(batch, n_heads, n_kv_heads, head_dim, capacity), 256);
    const size_t parts = (size_t)rows * n_kv_heads * (pl.splits + 1);
    pl.off_o = pl.off_ml + align_up(parts * 2 * sizeof(float), 256);
    pl.bytes = pl.off_o + align_up(parts * head_dim * sizeof(float), 256);
    return pl;
}

template <bool BF, int D>
void launch_prefix(const PagedFlashParams& f, const PagedDecodeParams& d, int flash_wgs, int decode_wgs, bool uniform,
                   hipStream_t stream) {
    const unsigned grid = (unsigned)(flash_wgs + decode_wgs);
    auto go = [&](auto uni, auto exact) {
        paged_prefix_kernel<BF, D, decltype(uni)::value, decltype(exact)::value>
            <<<grid, kPfThreads, 0, stream>>>(f, d, (uint32_t)flash_wgs);
    };
    using std::false_type;
    using std::true_type;
    if (f.s.cap_x != 0.0f) uniform ? go(true_type{}, true_type{}) : go(false_type{}, true_type{});
    else uniform ? go(true_type{}, false_type{}) : go(false_type{}, false_type{});
    const int rows = f.c.batch * f.n_heads, per_wg = 4 * 128 / D;
    paged_prefix_join_kernel<BF, D><<<(unsigned)((rows + per_wg - 1) / per_wg), 256, 0, stream>>>(
        f.part_o, f.part_ml, f.out, f.splits + 1, rows, FastDiv::of((uint32_t)(f.c.batch * d.gqa)), f.gqa);
}

}  // namespace

size_t paged_prefix_workspace(int batch, int n_heads, int n_kv_heads, int head_dim, long capacity, int prefix_len) {
    return plan_prefix(batch, n_heads, n_kv_heads, head_dim, capacity, prefix_len, device_cu_count()).bytes;
}

int launch_paged_shared_prefix(const PagedLaunch& a, hipStream_t stream) {
    const int cus = device_cu_count();
    const long capacity = std::min((long)a.max_pages * a.page_size, kMaxPagedTokens);
    const PagedPrefixPlan pl = plan_prefix(a.batch, a.n_heads, a.n_kv_heads, a.head_dim, capacity, a.prefix_len, cus);
    if (a.workspace == nullptr || a.workspace_bytes < pl.bytes)
        return set_error(LLMIK_ERR_WORKSPACE, "workspace too small (llmik_paged_workspace_size)");
    const PagedDecodePlan dp = plan_paged_decode(a.batch, a.n_heads, a.n_kv_heads, a.head_dim, capacity, cus);
    if ((long)dp.workgroups > kMaxCounters)
        return set_error(LLMIK_ERR_UNSUPPORTED, "too many compute units for the workspace's counters");
    char* ws = static_cast<char*>(a.workspace);
    PagedFlashParams f = flash_params(a);
    f.prefix_pages = a.prefix_pages;
    f.prefix_len = a.prefix_len;
    f.splits = pl.splits;
    f.chunk = pl.chunk;
    f.part_ml = reinterpret_cast<float*>(ws + pl.off_ml);
    f.part_o = reinterpret_cast<float*>(ws + pl.off_o);
    PagedDecodeParams d = paged_decode_params(a, dp);
    d.first = a.prefix_len;
    d.own_o = f.part_o;
    d.own_ml = f.part_ml;
    d.own_parts = pl.splits + 1;
    const long flash_wgs = (long)pl.row_tiles * pl.splits * a.n_kv_heads;
    const int decode_wgs = dp.workgroups;
    d.few_steps = decode_wgs;
    const bool uniform = a.page_size % 32 == 0;
    if (a.bf16)
        a.head_dim == 128 ? launch_prefix<true, 128>(f, d, (int)flash_wgs, decode_wgs, uniform, stream)
                          : launch_prefix<true, 64>(f, d, (int)flash_wgs, decode_wgs, uniform, stream);
    else
        a.head_dim == 128 ? launch_prefix<false, 128>(f, d, (int)flash_wgs, decode_wgs, uniform, stream)
                          : launch_prefix<false, 64>(f, d, (int)flash_wgs, decode_wgs, uniform, stream);
    return check_launch();
}

}  // namespace llmik
