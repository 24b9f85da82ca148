// extern "C" entry points of the paged KV cache (include/llmik.h): argument
// checks before any launch, as capi.cpp's.
#include <algorithm>
#include <climits>
#include <cmath>

#include "llmik_internal.hpp"

using namespace llmik;

namespace {

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
int invalid(const char* msg) { return set_error(LLMIK_ERR_INVALID, msg); }
int unsupported(const char* msg) { return set_error(LLMIK_ERR_UNSUPPORTED, msg); }
int misaligned(const char* msg) { return set_error(LLMIK_ERR_ALIGNMENT, msg); }

constexpr float kMaxSoftcap = 4096.0f;   // (as far as capped scores are tested)
// HIP launches hold fewer than 2^32 threads.
constexpr long kMaxThreads = (1L << 32) - 1;

long row_elements(const llmik_paged_cache& c) { return (long)c.page_size * c.head_dim * c.n_kv_heads; }
long page_stride(const llmik_paged_cache& c) { return c.page_stride ? (long)c.page_stride : row_elements(c); }

int check_shapes(const llmik_paged_cache* c, int n_heads) {
    if (c == nullptr) return invalid("null cache");
    if (c->head_dim != 64 && c->head_dim != 128) return invalid("only head_dim=64 and 128 supported");
    if (c->dtype != LLMIK_F16 && c->dtype != LLMIK_BF16) return invalid("dtype must be LLMIK_F16 or LLMIK_BF16");
    if (n_heads <= 0 || c->n_kv_heads <= 0) return invalid("head counts must be positive");
    if (n_heads % c->n_kv_heads != 0) return invalid("n_heads must be a multiple of n_kv_heads");
    if (c->page_size <= 0 || c->page_size % 8 != 0) return invalid("page_size must be a positive multiple of 8");
    if (c->page_size > (1 << 20) || c->n_kv_heads > (1 << 16) || n_heads > (1 << 16))
        return unsupported("page_size above 2^20 or more than 2^16 heads");
    if (c->n_pages <= 0) return invalid("the cache has no pages");
    if (c->batch < 0) return invalid("batch must be >= 0");
    if (c->max_pages <= 0) return invalid("page_table must have at least one column");
    if (page_stride(*c) < row_elements(*c) || page_stride(*c) % 8 != 0)
        return invalid("page_stride must hold a page and be a multiple of 8");
    // the work of all sequences is counted in 32 bits
    const long capacity = std::min((long)c->max_pages * c->page_size, kMaxPagedTokens);
    const long chunks = (n_heads / c->n_kv_heads + 15) / 16;
    const long slabs = (long)c->batch * c->n_kv_heads * chunks;
    if (slabs >= INT_MAX || slabs * ((capacity + 31) / 32 + kPieceUnits) >= INT_MAX)
        return unsupported("batch * n_kv_heads * page table capacity too large");
    return LLMIK_OK;
}

int check_cache(const llmik_paged_cache* c, int n_heads) {
    const int st = check_shapes(c, n_heads);
    if (st != LLMIK_OK || c->batch == 0) return st;
    if (!c->k || !c->v || !c->page_table || !c->seq_lens) return invalid("null cache pointer");
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return misaligned("k and v must be 16-byte aligned");
    if (!aligned(c->page_table, 4) || !aligned(c->seq_lens, 4))
        return misaligned("page_table and seq_lens must be 4-byte aligned");
    return LLMIK_OK;
}

int check_options(const llmik_score_options* o) {
    if (o == nullptr) return invalid("null score options");
    if (!std::isfinite(o->softmax_scale)) return invalid("softmax_scale must be finite");
    if (!(o->softcap >= 0.0f && o->softcap <= kMaxSoftcap)) return invalid("softcap must be >= 0 and at most 4096");
    if (o->softcap > 0.0f && !std::isfinite(4.0f * (o->softmax_scale / o->softcap)))
        return invalid("softcap too small for softmax_scale");
    if (o->window < 0) return invalid("window must be >= 0");
    if (!aligned(o->slopes, 4)) return misaligned("slopes must be 4-byte aligned");
    return LLMIK_OK;
}

// A ragged call's rows: its row tiles (of 128 rows per KV head) are counted in 32 bits.
int check_rows(const llmik_paged_cache* c, int n_heads, int rows) {
    const int st = check_shapes(c, n_heads);
    if (st != LLMIK_OK) return st;
    if (rows < 0) return invalid("rows must be >= 0");
    const long per_kv = (long)rows * (n_heads / c->n_kv_heads);
    if (per_kv >= INT_MAX - 256 || (per_kv / 128 + c->batch + 1) * c->n_kv_heads * 256 * 4 > kMaxThreads)
        return unsupported("too many rows");
    return LLMIK_OK;
}

// A shared-prefix call's sizes (those of a cache that check_shapes accepts).
int check_prefix(const llmik_paged_cache* c, int n_heads, int prefix_len) {
    if (prefix_len < 0) return invalid("prefix_len must be >= 0");
    if (prefix_len > kMaxPagedTokens) return unsupported("prefix_len too large");
    const long per_kv = (long)c->batch * (n_heads / c->n_kv_heads);
    if (prefix_len > 0 &&
        (per_kv >= INT_MAX - 256 || (per_kv / 128 + 1) * 64 * c->n_kv_heads * 256 > kMaxThreads))
        return unsupported("too many rows");
    return LLMIK_OK;
}

int check_q(const void* q, const void* out) {
    if (!q || !out) return invalid("null q/out pointer");
    if (!aligned(q, 16) || !aligned(out, 16)) return misaligned("q/out must be 16-byte aligned");
    return LLMIK_OK;
}

PagedLaunch launch_of(const llmik_paged_cache& c, const void* q, void* out, int n_heads,
                      const llmik_score_options& o) {
    PagedLaunch a{};
    a.q = q;
    a.k = c.k;
    a.v = c.v;
    a.out = out;
    a.table = c.page_table;
    a.lens = c.seq_lens;
    a.slopes = o.slopes;
    a.page_stride = page_stride(c);
    a.n_pages = c.n_pages;
    a.page_size = c.page_size;
    a.max_pages = c.max_pages;
    a.batch = c.batch;
    a.n_heads = n_heads;
    a.n_kv_heads = c.n_kv_heads;
    a.head_dim = c.head_dim;
    a.window = o.window;
    a.softmax_scale = o.softmax_scale;
    a.softcap = o.softcap;
    a.bf16 = c.dtype == LLMIK_BF16;
    return a;
}

long capacity_of(const llmik_paged_cache& c) {
    return std::min((long)c.max_pages * c.page_size, kMaxPagedTokens);
}

hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

}  // namespace

extern "C" {

LLMIK_API llmik_status llmik_rope_paged_append(const llmik_paged_cache* cache, const void* qkv, const void* cos,
                                               const void* sin, int table_rows, int table_f32, const int* cu_tokens,
                                               void* q_out, int rows, int n_heads, void* stream) {
    const int st = check_cache(cache, n_heads);
    if (st != LLMIK_OK) return st;
    if (rows < 0) return invalid("rows must be >= 0");
    if (cu_tokens == nullptr && rows != cache->batch)
        return invalid("without cu_tokens there is one row per sequence");
    if ((cos == nullptr) != (sin == nullptr)) return invalid("cos and sin come together");
    if (cos != nullptr && table_rows < 0) return invalid("table_rows must be >= 0");
    if (rows == 0) return LLMIK_OK;
    if (cache->batch == 0) return invalid("rows without a sequence");
    if (!qkv || !q_out) return invalid("null qkv/q_out pointer");
    if (!aligned(qkv, 16) || !aligned(q_out, 16) || !aligned(cos, 16) || !aligned(sin, 16))
        return misaligned("qkv, q_out, cos and sin must be 16-byte aligned");
    if (!aligned(cu_tokens, 4)) return misaligned("cu_tokens must be 4-byte aligned");
    const long threads = ((long)n_heads + 2L * cache->n_kv_heads) * (cache->head_dim / 16) + 1024;
    if (threads > 65535L * 64 || (long)rows * threads > kMaxThreads) return unsupported("too many rows or heads");
    PagedAppend a{};
    a.qkv = qkv;
    a.cos = cos;
    a.sin = sin;
    a.q_out = q_out;
    a.k = cache->k;
    a.v = cache->v;
    a.table = cache->page_table;
    a.lens = cache->seq_lens;
    a.cu = cu_tokens;
    a.page_stride = page_stride(*cache);
    a.n_pages = cache->n_pages;
    a.page_size = cache->page_size;
    a.max_pages = cache->max_pages;
    a.batch = cache->batch;
    a.n_heads = n_heads;
    a.n_kv_heads = cache->n_kv_heads;
    a.head_dim = cache->head_dim;
    a.rows = rows;
    a.table_rows = table_rows;
    a.bf16 = cache->dtype == LLMIK_BF16;
    a.table_f32 = table_f32 != 0;
    return launch_paged_append(a, as_stream(stream));
}

LLMIK_API size_t llmik_paged_workspace_size(const llmik_paged_cache* cache, int n_heads, int prefix_len) {
    if (check_shapes(cache, n_heads) != LLMIK_OK || cache->batch == 0) return 0;
    if (check_prefix(cache, n_heads, prefix_len) != LLMIK_OK) return 0;
    if (prefix_len > 0)
        return paged_prefix_workspace(cache->batch, n_heads, cache->n_kv_heads, cache->head_dim, capacity_of(*cache),
                                      prefix_len);
    return paged_decode_workspace(cache->batch, n_heads, cache->n_kv_heads, cache->head_dim, capacity_of(*cache));
}

LLMIK_API llmik_status llmik_paged_decode_attention(const llmik_paged_cache* cache, const void* q, void* out,
                                                    int n_heads, const llmik_score_options* options,
                                                    void* workspace, size_t workspace_bytes, void* stream) {
    int st = check_cache(cache, n_heads);
    if (st == LLMIK_OK) st = check_options(options);
    if (st != LLMIK_OK || cache->batch == 0) return st;
    if ((st = check_q(q, out)) != LLMIK_OK) return st;
    PagedLaunch a = launch_of(*cache, q, out, n_heads, *options);
    a.workspace = workspace;
    a.workspace_bytes = workspace_bytes;
    return launch_paged_decode(a, as_stream(stream));
}

LLMIK_API size_t llmik_paged_prefill_workspace_size(const llmik_paged_cache* cache, int n_heads, int rows) {
    if (check_rows(cache, n_heads, rows) != LLMIK_OK || cache->batch == 0 || rows == 0) return 0;
    return paged_prefill_workspace(cache->batch, rows, n_heads, cache->n_kv_heads, cache->head_dim,
                                   capacity_of(*cache));
}

LLMIK_API llmik_status llmik_paged_prefill_attention(const llmik_paged_cache* cache, const void* q,
                                                     const int* cu_tokens, void* out, int rows, int n_heads,
                                                     const llmik_score_options* options, void* workspace,
                                                     size_t workspace_bytes, void* stream) {
    int st = check_cache(cache, n_heads);
    if (st == LLMIK_OK) st = check_options(options);
    if (st == LLMIK_OK) st = check_rows(cache, n_heads, rows);
    if (st != LLMIK_OK) return st;
    if (rows == 0) return LLMIK_OK;
    if (cache->batch == 0) return invalid("rows without a sequence");
    if (cu_tokens == nullptr) return invalid("null cu_tokens pointer");
    if (!aligned(cu_tokens, 4)) return misaligned("cu_tokens must be 4-byte aligned");
    if ((st = check_q(q, out)) != LLMIK_OK) return st;
    PagedLaunch a = launch_of(*cache, q, out, n_heads, *options);
    a.cu = cu_tokens;
    a.rows = rows;
    a.workspace = workspace;
    a.workspace_bytes = workspace_bytes;
    return launch_paged_prefill(a, as_stream(stream));
}

LLMIK_API llmik_status llmik_paged_shared_prefix_attention(const llmik_paged_cache* cache, const void* q, void* out,
                                                           int n_heads, const int* prefix_pages, int n_prefix_pages,
                                                           int prefix_len, const llmik_score_options* options,
                                                           void* workspace, size_t workspace_bytes, void* stream) {
    int st = check_cache(cache, n_heads);
    if (st == LLMIK_OK) st = check_options(options);
    if (st == LLMIK_OK) st = check_prefix(cache, n_heads, prefix_len);
    if (st != LLMIK_OK || cache->batch == 0) return st;
    if ((st = check_q(q, out)) != LLMIK_OK) return st;
    if ((long)n_prefix_pages * cache->page_size < prefix_len)
        return invalid("prefix_pages hold fewer than prefix_len tokens");
    PagedLaunch a = launch_of(*cache, q, out, n_heads, *options);
    a.workspace = workspace;
    a.workspace_bytes = workspace_bytes;
    if (prefix_len == 0) return launch_paged_decode(a, as_stream(stream));
    if (prefix_pages == nullptr) return invalid("null prefix_pages pointer");
    if (!aligned(prefix_pages, 4)) return misaligned("prefix_pages must be 4-byte aligned");
    a.prefix_pages = prefix_pages;
    a.prefix_len = prefix_len;
    a.rows = cache->batch;
    return launch_paged_shared_prefix(a, as_stream(stream));
}

}  // extern "C"
