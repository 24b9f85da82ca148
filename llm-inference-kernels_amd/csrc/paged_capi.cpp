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

int check_cache(const llmik_paged_cache* c, int n_heads, bool with_v = true) {
    const int st = check_shapes(c, n_heads);
    if (st != LLMIK_OK || c->batch == 0) return st;
    if (!c->k || (with_v && !c->v) || !c->page_table || !c->seq_lens) return invalid("null cache pointer");
    if (!aligned(c->k, 16) || (with_v && !aligned(c->v, 16))) return misaligned("k and v must be 16-byte aligned");
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

// A call whose row tiles' keys are cut by length counts pairs of both kinds of tiles in 32 bits.
int check_cut(const llmik_paged_cache* c, int n_heads, int rows) {
    const int st = check_rows(c, n_heads, rows);
    if (st != LLMIK_OK) return st;
    const long capacity = std::min((long)c->max_pages * c->page_size, kMaxPagedTokens);
    const long per_kv = (long)rows * (n_heads / c->n_kv_heads);
    if ((per_kv / 64 + c->batch + 1) * (capacity / 64 + 2) >= INT_MAX)
        return unsupported("rows * page table capacity too large");
    return LLMIK_OK;
}

int check_weights(const llmik_token_weights* w, int batch) {
    if (w == nullptr) return invalid("null token weights");
    if (w->n_rows < 0) return invalid("n_rows must be >= 0");
    if (w->max_len <= 0 || w->max_len > kMaxPagedTokens) return invalid("max_len must be positive and at most 2^30");
    if (w->rows == nullptr && w->n_rows < batch) return invalid("without rows there is one row per sequence");
    if (w->weights == nullptr && w->n_rows > 0) return invalid("null weights pointer");
    if (!aligned(w->weights, 4) || !aligned(w->rows, 4)) return misaligned("weights and rows must be 4-byte aligned");
    return LLMIK_OK;
}

PagedWeights weights_of(const llmik_token_weights& w) { return {w.weights, w.rows, w.n_rows, w.max_len}; }

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
    return llmik_rope_paged_append_at(cache, qkv, cos, sin, table_rows, table_f32, cu_tokens, nullptr, q_out, rows,
                                      n_heads, stream);
}

LLMIK_API llmik_status llmik_rope_paged_append_at(const llmik_paged_cache* cache, const void* qkv, const void* cos,
                                                  const void* sin, int table_rows, int table_f32,
                                                  const int* cu_tokens, const int* positions, void* q_out, int rows,
                                                  int n_heads, void* stream) {
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
    if (!aligned(positions, 4)) return misaligned("positions must be 4-byte aligned");
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
    a.positions = positions;
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

LLMIK_API size_t llmik_paged_tree_workspace_size(const llmik_paged_cache* cache, int n_heads, int rows) {
    if (check_cut(cache, n_heads, rows) != LLMIK_OK || cache->batch == 0 || rows == 0) return 0;
    return paged_tree_workspace(cache->batch, rows, n_heads, cache->n_kv_heads, cache->head_dim,
                                capacity_of(*cache));
}

LLMIK_API llmik_status llmik_paged_tree_attention(const llmik_paged_cache* cache, const void* q,
                                                  const int* cu_tokens, const uint64_t* tree_mask, int words,
                                                  const int* positions, void* out, int rows, int n_heads,
                                                  const llmik_score_options* options, void* workspace,
                                                  size_t workspace_bytes, void* stream) {
    int st = check_cache(cache, n_heads);
    if (st == LLMIK_OK) st = check_options(options);
    if (st == LLMIK_OK) st = check_cut(cache, n_heads, rows);
    if (st != LLMIK_OK) return st;
    if (words <= 0) return invalid("tree_mask must have at least one word per row");
    if (words > (1 << 24)) return unsupported("tree_mask has more than 2^24 words per row");
    if (rows == 0) return LLMIK_OK;
    if (cache->batch == 0) return invalid("rows without a sequence");
    if (cu_tokens == nullptr || tree_mask == nullptr) return invalid("null cu_tokens/tree_mask pointer");
    if (!aligned(cu_tokens, 4) || !aligned(positions, 4))
        return misaligned("cu_tokens and positions must be 4-byte aligned");
    if (!aligned(tree_mask, 8)) return misaligned("tree_mask must be 8-byte aligned");
    if ((st = check_q(q, out)) != LLMIK_OK) return st;
    PagedLaunch a = launch_of(*cache, q, out, n_heads, *options);
    a.cu = cu_tokens;
    a.rows = rows;
    a.workspace = workspace;
    a.workspace_bytes = workspace_bytes;
    return launch_paged_tree(a, tree_mask, words, positions, as_stream(stream));
}

LLMIK_API size_t llmik_paged_decode_weights_scratch_size(const llmik_paged_cache* cache, int n_heads,
                                                         const llmik_token_weights* weights) {
    if (check_shapes(cache, n_heads) != LLMIK_OK || cache->batch == 0) return 0;
    if (check_weights(weights, cache->batch) != LLMIK_OK) return 0;
    return paged_decode_weights_scratch(cache->batch, n_heads, capacity_of(*cache), weights->max_len);
}

LLMIK_API llmik_status llmik_paged_decode_attention_weights(const llmik_paged_cache* cache, const void* q, void* out,
                                                            int n_heads, const llmik_score_options* options,
                                                            const llmik_token_weights* weights, void* scratch,
                                                            size_t scratch_bytes, void* workspace,
                                                            size_t workspace_bytes, void* stream) {
    int st = check_cache(cache, n_heads);
    if (st == LLMIK_OK) st = check_options(options);
    if (st == LLMIK_OK) st = check_weights(weights, cache->batch);
    if (st != LLMIK_OK || cache->batch == 0) return st;
    if ((st = check_q(q, out)) != LLMIK_OK) return st;
    if (!aligned(scratch, 16)) return misaligned("scratch must be 16-byte aligned");
    PagedLaunch a = launch_of(*cache, q, out, n_heads, *options);
    a.workspace = workspace;
    a.workspace_bytes = workspace_bytes;
    return launch_paged_decode_weights(a, weights_of(*weights), scratch, scratch_bytes, as_stream(stream));
}

LLMIK_API size_t llmik_paged_prefill_weights_workspace_size(const llmik_paged_cache* cache, int n_heads, int rows,
                                                            int observe) {
    if (check_cut(cache, n_heads, rows) != LLMIK_OK || cache->batch == 0 || rows == 0 || observe < 0) return 0;
    return paged_prefill_weights_workspace(cache->batch, rows, n_heads, cache->n_kv_heads, observe);
}

LLMIK_API llmik_status llmik_paged_prefill_weights(const llmik_paged_cache* cache, const void* q,
                                                   const int* cu_tokens, int rows, int n_heads,
                                                   const llmik_score_options* options, int observe,
                                                   const llmik_token_weights* weights, void* workspace,
                                                   size_t workspace_bytes, void* stream) {
    int st = check_cache(cache, n_heads, false);
    if (st == LLMIK_OK) st = check_options(options);
    if (st == LLMIK_OK) st = check_cut(cache, n_heads, rows);
    if (st == LLMIK_OK) st = check_weights(weights, cache->batch);
    if (st != LLMIK_OK) return st;
    if (observe < 0) return invalid("observe must be >= 0");
    if (rows == 0) return LLMIK_OK;
    if (cache->batch == 0) return invalid("rows without a sequence");
    if (cu_tokens == nullptr) return invalid("null cu_tokens pointer");
    if (!aligned(cu_tokens, 4)) return misaligned("cu_tokens must be 4-byte aligned");
    if (q == nullptr) return invalid("null q pointer");
    if (!aligned(q, 16)) return misaligned("q must be 16-byte aligned");
    PagedLaunch a = launch_of(*cache, q, nullptr, n_heads, *options);
    a.cu = cu_tokens;
    a.rows = rows;
    a.workspace = workspace;
    a.workspace_bytes = workspace_bytes;
    return launch_paged_prefill_weights(a, weights_of(*weights), observe, as_stream(stream));
}

LLMIK_API llmik_status llmik_paged_select_tokens(const llmik_token_weights* weights, const int* seq_lens, int batch,
                                                 int n_kv_heads, int keep, int first, int recent, int* kept,
                                                 int* new_lens, void* stream) {
    if (batch < 0) return invalid("batch must be >= 0");
    if (n_kv_heads <= 0) return invalid("head counts must be positive");
    const int st = check_weights(weights, batch);
    if (st != LLMIK_OK) return st;
    if (keep <= 0) return invalid("keep must be positive");
    if (first < 0 || recent < 0 || (long)first + recent > keep)
        return invalid("first and recent must be >= 0, together at most keep");
    if (batch == 0) return LLMIK_OK;
    if (!seq_lens || !kept || !new_lens) return invalid("null seq_lens/kept/new_lens pointer");
    if (!aligned(seq_lens, 4) || !aligned(kept, 4) || !aligned(new_lens, 4))
        return misaligned("seq_lens, kept and new_lens must be 4-byte aligned");
    if ((long)batch * n_kv_heads * 1024 > kMaxThreads) return unsupported("batch * n_kv_heads too large");
    return launch_paged_select(weights_of(*weights), seq_lens, batch, n_kv_heads, keep, first, recent, kept, new_lens,
                               as_stream(stream));
}

LLMIK_API llmik_status llmik_paged_compact(const llmik_paged_cache* cache, const int* kept, int kept_heads, int n,
                                           const int* starts, const llmik_token_weights* weights, void* stream) {
    int st = check_cache(cache, cache != nullptr ? cache->n_kv_heads : 1);
    if (st == LLMIK_OK && weights != nullptr) st = check_weights(weights, cache->batch);
    if (st != LLMIK_OK) return st;
    if (kept_heads != 1 && kept_heads != cache->n_kv_heads) return invalid("kept_heads must be 1 or n_kv_heads");
    if (n < 0) return invalid("n must be >= 0");
    if (n > kMaxPagedTokens) return unsupported("n too large");
    if (cache->batch == 0) return LLMIK_OK;
    if (kept == nullptr && n > 0) return invalid("null kept pointer");
    if (!aligned(kept, 4) || !aligned(starts, 4)) return misaligned("kept and starts must be 4-byte aligned");
    if ((long)cache->batch * cache->n_kv_heads * 16 * 1024 > kMaxThreads)
        return unsupported("batch * n_kv_heads too large");
    const PagedLaunch a = launch_of(*cache, nullptr, nullptr, cache->n_kv_heads, llmik_score_options{});
    const PagedWeights w = weights != nullptr ? weights_of(*weights) : PagedWeights{};
    return launch_paged_compact(a, w, kept, kept_heads, n, starts, as_stream(stream));
}

}  // extern "C"
