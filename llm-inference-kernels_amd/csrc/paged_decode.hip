// Decode attention over a paged cache (paged_decode.hpp): its launches.
#include "paged_decode.hpp"

namespace llmik {

template <bool BF, int D, bool UNI, bool EXACT>
__global__ __launch_bounds__(kPdThreads, kPdPerCu) void paged_decode_kernel(PagedDecodeParams p) {
    constexpr int kFloats = DecodeLds<D>::kFloats;
    __shared__ __attribute__((aligned(16))) float s_o[kPdWaves * kFloats];
    __shared__ float s_m[kPdWaves][16], s_l[kPdWaves][16];
    __shared__ uint32_t s_last;
    paged_decode<BF, D, UNI, EXACT>(p, blockIdx.x, gridDim.x,
                                    {s_o, s_o + kFloats, s_o + 2 * kFloats, s_o + 3 * kFloats, s_m, s_l, &s_last});
}

namespace {

template <bool BF, int D>
void launch_decode(const PagedDecodeParams& p, int workgroups, bool uniform, hipStream_t stream) {
    auto go = [&](auto uni, auto exact) {
        paged_decode_kernel<BF, D, decltype(uni)::value, decltype(exact)::value>
            <<<workgroups, kPdThreads, 0, stream>>>(p);
    };
    using std::false_type;
    using std::true_type;
    if (p.s.cap_x != 0.0f) uniform ? go(true_type{}, true_type{}) : go(false_type{}, true_type{});
    else uniform ? go(true_type{}, false_type{}) : go(false_type{}, false_type{});
}

}  // namespace

size_t paged_decode_workspace(int batch, int n_heads, int n_kv_heads, int head_dim, long capacity) {
    return plan_paged_decode(batch, n_heads, n_kv_heads, head_dim, capacity, device_cu_count()).bytes;
}

int launch_paged_decode(const PagedLaunch& a, hipStream_t stream) {
    const long capacity = std::min((long)a.max_pages * a.page_size, kMaxPagedTokens);
    const PagedDecodePlan pl =
        plan_paged_decode(a.batch, a.n_heads, a.n_kv_heads, a.head_dim, capacity, device_cu_count());
    if (a.workspace == nullptr || a.workspace_bytes < pl.bytes)
        return set_error(LLMIK_ERR_WORKSPACE, "workspace too small (llmik_paged_workspace_size)");
    if ((long)pl.workgroups > kMaxCounters)
        return set_error(LLMIK_ERR_UNSUPPORTED, "too many compute units for the workspace's counters");
    const PagedDecodeParams p = paged_decode_params(a, pl);
    const bool uniform = a.page_size % 32 == 0;
    if (a.bf16)
        a.head_dim == 128 ? launch_decode<true, 128>(p, pl.workgroups, uniform, stream)
                          : launch_decode<true, 64>(p, pl.workgroups, uniform, stream);
    else
        a.head_dim == 128 ? launch_decode<false, 128>(p, pl.workgroups, uniform, stream)
                          : launch_decode<false, 64>(p, pl.workgroups, uniform, stream);
    return check_launch();
}

}  // namespace llmik
