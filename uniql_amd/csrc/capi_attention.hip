// extern "C" surface of the 4-bit key / value cache and of attention: argument checks and dispatch.  Nothing here allocates,
// synchronises or throws.
#include "kv_attention.hpp"
#include "prompt_attention.hpp"

namespace uniql {
int kv_assign_launch(const int32_t* new_tokens, const int32_t* lengths, int32_t* table, int32_t* free_pages, const int32_t* free_count,
                     int32_t* lengths_out, int32_t* free_count_out, int64_t* slots, int32_t* positions, int32_t* cu, int32_t* refused,
                     int rows, int columns, int pool, int page_size, int max_tokens, hipStream_t stream);
int kv4_store_launch(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const int64_t* slots,
                     const KvCache& cache, int tokens, hipStream_t stream);
int kv4_load_launch(const KvCache& cache, const int32_t* table, const int32_t* cu, const int32_t* starts, void* k, int64_t k_row,
                    int64_t k_head, void* v, int64_t v_row, int64_t v_head, int requests, int columns, int rows, hipStream_t stream);
void kv4_attention_needs(int rows, int requests, int q_heads, const KvCache& cache, size_t* accum_bytes, size_t* temp_bytes);
int kv4_attention_launch(const KvAttentionArgs& a, hipStream_t stream);
int prompt_attention_launch(const PromptArgs& a, hipStream_t stream);
}  // namespace uniql

using namespace uniql;

static constexpr int kMaxHeads = 4096, kMaxWidth = 128;
// requests or sequences: sums of two of their numbers, and steps beyond the last, stay below 2^31
static constexpr int kMaxRequests = 1 << 30;

// Scales up to 2^64: finite queries and keys (128 products of 2^32) then have finite scores, also with the factors that the
// kernels fold into the scale.
static bool scale_ok(float v) { return v >= -18446744073709551616.0f && v <= 18446744073709551616.0f; }
static bool page_size_ok(int n) { return n == 16 || n == 32 || n == 64 || n == 128 || n == 256; }
// rows and columns of a table, and the tokens that a row of it has room for
static bool columns_ok(int64_t rows, int64_t columns, int64_t page_size) {
    return rows <= kMaxRequests && columns > 0 && columns <= (1 << 20) && columns * page_size <= (1LL << 30) && rows * columns <= 0x7fffffffLL;
}

// Sizes first, then (when there is work to do) pointers.
static int cache_sizes(const uniql_kv4_cache* c, KvCache& out) {
    if (!c) return UNIQL_E_NULL;
    if (!page_size_ok(c->page_size) || c->pages <= 0 || c->heads <= 0 || c->heads > kMaxHeads) return UNIQL_E_SHAPE;
    if (c->k_dim <= 0 || c->v_dim <= 0) return UNIQL_E_SHAPE;
    if (c->k_dim > kMaxWidth || c->v_dim > kMaxWidth) return UNIQL_E_UNSUPPORTED;
    out.k_codes = reinterpret_cast<uint32_t*>(c->k_codes);
    out.v_codes = reinterpret_cast<uint32_t*>(c->v_codes);
    out.k_scales = reinterpret_cast<half_t*>(c->k_scales);
    out.v_scales = reinterpret_cast<half_t*>(c->v_scales);
    out.pages = c->pages;
    out.page_shift = __builtin_ctz((unsigned)c->page_size);
    out.heads = c->heads;
    out.k_dim = c->k_dim;
    out.v_dim = c->v_dim;
    out.k_words = 4 * ((c->k_dim + 31) / 32);
    out.v_words = 4 * ((c->v_dim + 31) / 32);
    return UNIQL_OK;
}
static int cache_pointers(const KvCache& c) {
    if (!c.k_codes || !c.v_codes || !c.k_scales || !c.v_scales) return UNIQL_E_NULL;
    const uintptr_t all = reinterpret_cast<uintptr_t>(c.k_codes) | reinterpret_cast<uintptr_t>(c.v_codes) |
                          reinterpret_cast<uintptr_t>(c.k_scales) | reinterpret_cast<uintptr_t>(c.v_scales);
    return (all & 15u) ? UNIQL_E_ALIGN : UNIQL_OK;
}

extern "C" {

int uniql_kv_assign_pages(const int32_t* new_tokens, const int32_t* lengths, int32_t* table, int32_t* free_pages,
                          const int32_t* free_count, int32_t* lengths_out, int32_t* free_count_out, int64_t* slots, int32_t* positions,
                          int32_t* cu, int32_t* refused, int rows, int columns, int pool, int page_size, int max_tokens, void* stream) {
    if (rows < 0 || pool < 0 || max_tokens < 0 || max_tokens > (1 << 24) || !page_size_ok(page_size) ||
        !columns_ok(rows, columns, page_size))
        return UNIQL_E_SHAPE;
    if (!free_count || !free_count_out || !cu) return UNIQL_E_NULL;
    if (rows > 0 && (!new_tokens || !lengths || !table || !lengths_out || !refused)) return UNIQL_E_NULL;
    if ((pool > 0 && !free_pages) || (max_tokens > 0 && (!slots || !positions))) return UNIQL_E_NULL;
    return kv_assign_launch(new_tokens, lengths, table, free_pages, free_count, lengths_out, free_count_out, slots, positions, cu, refused,
                            rows, columns, pool, page_size, max_tokens, reinterpret_cast<hipStream_t>(stream));
}

int uniql_kv4_store(const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const int64_t* slots,
                    const uniql_kv4_cache* cache, int tokens, void* stream) {
    KvCache c;
    if (const int code = cache_sizes(cache, c)) return code;
    if (tokens < 0 || tokens > (1 << 27)) return UNIQL_E_SHAPE;
    if (tokens == 0) return UNIQL_OK;
    if (!k || !v || !slots) return UNIQL_E_NULL;
    if (const int code = cache_pointers(c)) return code;
    return kv4_store_launch(k, k_row, k_head, v, v_row, v_head, slots, c, tokens, reinterpret_cast<hipStream_t>(stream));
}

int uniql_kv4_load(const uniql_kv4_cache* cache, const int32_t* table, const int32_t* cu, const int32_t* starts, void* k, int64_t k_row,
                   int64_t k_head, void* v, int64_t v_row, int64_t v_head, int requests, int columns, int rows, void* stream) {
    KvCache c;
    if (const int code = cache_sizes(cache, c)) return code;
    if (rows < 0 || rows > (1 << 27) || requests < 0 || !columns_ok(requests, columns, cache->page_size)) return UNIQL_E_SHAPE;
    if (rows == 0 || requests == 0) return UNIQL_OK;
    if (!table || !cu || !k || !v) return UNIQL_E_NULL;
    if (const int code = cache_pointers(c)) return code;
    return kv4_load_launch(c, table, cu, starts, k, k_row, k_head, v, v_row, v_head, requests, columns, rows,
                           reinterpret_cast<hipStream_t>(stream));
}

static int attention_sizes(const uniql_kv4_cache* cache, KvCache& c, int rows, int requests, int columns, int n_q_heads) {
    if (const int code = cache_sizes(cache, c)) return code;
    if (rows < 0 || requests < 0 || !columns_ok(requests, columns, cache->page_size)) return UNIQL_E_SHAPE;
    if (n_q_heads <= 0 || n_q_heads > kMaxHeads || n_q_heads % c.heads != 0) return UNIQL_E_SHAPE;
    if ((int64_t)rows * (n_q_heads / c.heads) > (1LL << 30)) return UNIQL_E_SHAPE;
    return UNIQL_OK;
}

int uniql_kv4_attention_workspace(const uniql_kv4_cache* cache, int rows, int requests, int columns, int n_q_heads, size_t* accum_bytes,
                                  size_t* temp_bytes) {
    if (!accum_bytes || !temp_bytes) return UNIQL_E_NULL;
    KvCache c;
    if (const int code = attention_sizes(cache, c, rows, requests, columns, n_q_heads)) return code;
    kv4_attention_needs(rows, requests, n_q_heads, c, accum_bytes, temp_bytes);
    return UNIQL_OK;
}

int uniql_kv4_attention(const void* q, int64_t q_row, int64_t q_head, const uniql_kv4_cache* cache, const int32_t* table,
                        const int32_t* lengths, const int32_t* cu_q, void* out, int64_t out_row, int64_t out_head, void* accum,
                        size_t accum_bytes, void* temp, size_t temp_bytes, int rows, int requests, int columns, int n_q_heads,
                        float scale, void* stream) {
    KvAttentionArgs a;
    if (const int code = attention_sizes(cache, a.cache, rows, requests, columns, n_q_heads)) return code;
    if (!scale_ok(scale)) return UNIQL_E_UNSUPPORTED;
    if (!cu_q && rows != requests) return UNIQL_E_SHAPE;
    if (rows == 0 || requests == 0) return UNIQL_OK;
    if (!q || !table || !lengths || !out) return UNIQL_E_NULL;
    if (const int code = cache_pointers(a.cache)) return code;
    size_t need_accum, need_temp;
    kv4_attention_needs(rows, requests, n_q_heads, a.cache, &need_accum, &need_temp);
    if (accum_bytes < need_accum || temp_bytes < need_temp) return UNIQL_E_WORKSPACE;
    if ((need_accum && !accum) || (need_temp && !temp)) return UNIQL_E_NULL;
    a.q = reinterpret_cast<const half_t*>(q);
    a.q_row = q_row;
    a.q_head = q_head;
    a.table = table;
    a.lengths = lengths;
    a.cu_q = cu_q;
    a.out = reinterpret_cast<half_t*>(out);
    a.out_row = out_row;
    a.out_head = out_head;
    a.accum = accum;
    a.temp = reinterpret_cast<float*>(temp);
    a.rows = rows;
    a.requests = requests;
    a.columns = columns;
    a.group = n_q_heads / a.cache.heads;
    a.scale = scale;
    return kv4_attention_launch(a, reinterpret_cast<hipStream_t>(stream));
}

int uniql_prompt_attention(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v,
                           int64_t v_row, int64_t v_head, const int32_t* cu_q, const int32_t* cu_k, void* out, int64_t out_row,
                           int64_t out_head, int rows, int k_rows, int sequences, int n_q_heads, int n_kv_heads, int k_dim, int v_dim,
                           int causal, float scale, void* stream) {
    if (rows < 0 || k_rows < 0 || sequences < 0 || n_kv_heads <= 0 || n_q_heads <= 0 || n_q_heads > kMaxHeads ||
        n_q_heads % n_kv_heads != 0 || k_dim <= 0 || v_dim <= 0 || sequences > kMaxRequests)
        return UNIQL_E_SHAPE;
    if (k_dim > kMaxWidth || v_dim > kMaxWidth || !scale_ok(scale)) return UNIQL_E_UNSUPPORTED;
    if (rows == 0 || sequences == 0) return UNIQL_OK;
    if (!q || !cu_q || !cu_k || !out || (k_rows > 0 && (!k || !v))) return UNIQL_E_NULL;
    PromptArgs a;
    a.q = reinterpret_cast<const half_t*>(q);
    a.k = reinterpret_cast<const half_t*>(k);
    a.v = reinterpret_cast<const half_t*>(v);
    a.out = reinterpret_cast<half_t*>(out);
    a.q_row = q_row, a.q_head = q_head, a.k_row = k_row, a.k_head = k_head, a.v_row = v_row, a.v_head = v_head;
    a.out_row = out_row, a.out_head = out_head;
    a.cu_q = cu_q, a.cu_k = cu_k;
    a.rows = rows, a.k_rows = k_rows, a.sequences = sequences;
    a.heads = n_q_heads, a.group = n_q_heads / n_kv_heads;
    a.k_dim = k_dim, a.v_dim = v_dim, a.causal = causal != 0;
    a.scale = scale;
    return prompt_attention_launch(a, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
