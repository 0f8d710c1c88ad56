// attn_api.cu -- the C entry points of the packed-prompt and paged-cache
// attention and of the cache's pages (include/rac_b200.h section 4).
#include <cstdio>

#include "attn_ops.h"
#include "rac_b200.h"
#include "rac_internal.h"

#define RAC_API extern "C" __attribute__((visibility("default")))

namespace {

using namespace racb;

int record(int st, const char* name) {
    if (st == kOk) return record_status(kOk, "ok");
    const char* kind = st == kErrNullPtr ? "null pointer" : st == kErrInvalidDim ? "invalid dimension"
                     : st == kErrAlloc ? "workspace too small" : st == kErrCuda ? "CUDA error"
                     : st == kErrUnsupported ? "unsupported head size, type or alignment" : "error";
    char msg[256];
    const cudaError_t ce = st == kErrCuda ? cudaGetLastError() : cudaSuccess;
    std::snprintf(msg, sizeof msg, "%s: %s%s%s", name, kind, ce != cudaSuccess ? " / " : "",
                  ce != cudaSuccess ? cudaGetErrorString(ce) : "");
    return record_status(st, msg);
}

PackedParams packed(const void* q, const void* k, const void* v, const long long* strides, const int* cu, int n_seqs,
                    long long tokens, int heads, int kv_heads, int head_dim, int dtype, int is_causal, float scale) {
    PackedParams p{};
    p.q = {q, strides[0], strides[1]};
    p.k = {k, strides[2], strides[3]};
    p.v = {v, strides[4], strides[5]};
    p.cu = cu; p.n_seqs = n_seqs; p.tokens = tokens;
    p.heads = heads; p.kv_heads = kv_heads; p.head_dim = head_dim;
    p.type = dtype; p.causal = is_causal; p.scale = scale;
    return p;
}

Pages pages(void* p, const long long* s) { return {p, s[1], s[2], s[3], s[0]}; }

}  // namespace

RAC_API long long rac_attention_packed_workspace(long long tokens, int n_seqs, int heads, int kv_heads, int head_dim,
                                                 int dtype, int backward) {
    if (tokens <= 0 || n_seqs < 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 0;
    return (long long)attention_packed_workspace(tokens, n_seqs, heads, kv_heads, head_dim, dtype, backward);
}

RAC_API int rac_attention_packed_async(const void* q, const void* k, const void* v, const long long* strides,
                                       const int* cu_seqlens, int n_seqs, long long tokens, int heads, int kv_heads,
                                       int head_dim, int dtype, int is_causal, float scale, void* out, float* lse,
                                       int zero_rest, void* workspace, long long ws_bytes, void* stream) {
    if (!strides) return record(kErrNullPtr, "rac_attention_packed_async");
    PackedParams p = packed(q, k, v, strides, cu_seqlens, n_seqs, tokens, heads, kv_heads, head_dim, dtype, is_causal,
                            scale);
    p.out = out; p.lse = lse; p.zero_rest = zero_rest;
    p.ws = workspace; p.ws_bytes = ws_bytes > 0 ? (size_t)ws_bytes : 0;
    return record(attention_packed(p, static_cast<cudaStream_t>(stream)), "rac_attention_packed_async");
}

RAC_API int rac_attention_packed_backward_async(const void* dout, const void* q, const void* k, const void* v,
                                                const long long* strides, const void* out, const float* lse,
                                                const int* cu_seqlens, int n_seqs, long long tokens, int heads,
                                                int kv_heads, int head_dim, int dtype, int is_causal, float scale,
                                                void* dq, void* dk, void* dv, void* workspace, long long ws_bytes,
                                                void* stream) {
    if (!strides) return record(kErrNullPtr, "rac_attention_packed_backward_async");
    PackedParams p = packed(q, k, v, strides, cu_seqlens, n_seqs, tokens, heads, kv_heads, head_dim, dtype, is_causal,
                            scale);
    p.dout = {dout, strides[6], strides[7]};
    p.out_in = out; p.lse_in = lse;
    p.dq = dq; p.dk = dk; p.dv = dv;
    p.ws = workspace; p.ws_bytes = ws_bytes > 0 ? (size_t)ws_bytes : 0;
    return record(attention_packed_backward(p, static_cast<cudaStream_t>(stream)),
                  "rac_attention_packed_backward_async");
}

RAC_API long long rac_attention_cached_workspace(int batch, int nodes, int heads, int kv_heads, int head_dim) {
    if (batch <= 0 || nodes <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 0;
    return (long long)attention_cached_workspace(batch, nodes, heads, kv_heads, head_dim);
}

RAC_API int rac_attention_cached_async(const void* q, const void* k_pages, const void* v_pages,
                                       const long long* strides, const int* page_table, int table_width, int n_pages,
                                       int page_size, const int* lengths, const int* counts, const long long* tree,
                                       int batch, int nodes, int heads, int kv_heads, int head_dim, int dtype,
                                       float scale, void* out, int zero_rest, void* workspace, long long ws_bytes,
                                       void* stream) {
    if (!strides) return record(kErrNullPtr, "rac_attention_cached_async");
    CachedParams p{};
    p.q = q; p.q_batch = strides[0]; p.q_node = strides[1]; p.q_head = strides[2];
    p.k = {const_cast<void*>(k_pages), strides[3], strides[4], strides[5], 0};
    p.v = {const_cast<void*>(v_pages), strides[6], strides[7], strides[8], 0};
    p.table = page_table; p.table_width = table_width; p.pages = n_pages; p.page_size = page_size;
    p.lengths = lengths; p.counts = counts; p.tree = tree;
    p.batch = batch; p.nodes = nodes; p.heads = heads; p.kv_heads = kv_heads; p.head_dim = head_dim; p.type = dtype;
    p.scale = scale; p.out = out; p.zero_rest = zero_rest;
    p.ws = workspace; p.ws_bytes = ws_bytes > 0 ? (size_t)ws_bytes : 0;
    return record(attention_cached(p, static_cast<cudaStream_t>(stream)), "rac_attention_cached_async");
}

RAC_API int rac_cache_append_async(void* k_pages, void* v_pages, const long long* strides, const void* k,
                                   const void* v, const int* page_table, int table_width, int n_pages, int page_size,
                                   const int* starts, const int* cu_seqlens, int batch, long long tokens,
                                   int kv_heads, int head_dim, int dtype, void* stream) {
    if (!strides) return record(kErrNullPtr, "rac_cache_append_async");
    AppendParams p{};
    p.k = pages(k_pages, strides); p.v = pages(v_pages, strides + 4);
    p.nk = {k, strides[8], strides[9]}; p.nv = {v, strides[10], strides[11]};
    p.table = page_table; p.table_width = table_width; p.pages = n_pages; p.page_size = page_size;
    p.starts = starts; p.cu = cu_seqlens; p.batch = batch; p.tokens = tokens;
    p.kv_heads = kv_heads; p.head_dim = head_dim; p.type = dtype;
    return record(cache_append(p, static_cast<cudaStream_t>(stream)), "rac_cache_append_async");
}

RAC_API int rac_cache_copy_pages_async(void* k_pages, void* v_pages, const long long* strides, const int* src,
                                       const int* dst, int n, int layers, int n_pages, int page_size, int kv_heads,
                                       int head_dim, int dtype, void* stream) {
    if (!strides) return record(kErrNullPtr, "rac_cache_copy_pages_async");
    CopyPagesParams p{};
    p.k = pages(k_pages, strides); p.v = pages(v_pages, strides + 4);
    p.src = src; p.dst = dst; p.n = n; p.layers = layers; p.pages = n_pages; p.page_size = page_size;
    p.kv_heads = kv_heads; p.head_dim = head_dim; p.type = dtype;
    return record(cache_copy_pages(p, static_cast<cudaStream_t>(stream)), "rac_cache_copy_pages_async");
}

RAC_API int rac_cache_compact_async(void* k_pages, void* v_pages, const long long* strides, const int* page_table,
                                    int table_width, int n_pages, int page_size, const int* starts,
                                    const int* accepted, const int* n_accepted, int batch, int nodes, int layers,
                                    int kv_heads, int head_dim, int dtype, void* stream) {
    if (!strides) return record(kErrNullPtr, "rac_cache_compact_async");
    CompactParams p{};
    p.k = pages(k_pages, strides); p.v = pages(v_pages, strides + 4);
    p.table = page_table; p.table_width = table_width; p.pages = n_pages; p.page_size = page_size;
    p.starts = starts; p.accepted = accepted; p.n_accepted = n_accepted; p.batch = batch; p.nodes = nodes;
    p.layers = layers; p.kv_heads = kv_heads; p.head_dim = head_dim; p.type = dtype;
    return record(cache_compact(p, static_cast<cudaStream_t>(stream)), "rac_cache_compact_async");
}
