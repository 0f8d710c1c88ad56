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

PackedParams packed(const rac_attention_packed_args& a) {
    PackedParams p{};
    const long long* st = a.strides;
    p.q = {a.q, st[0], st[1]};
    p.k = {a.k, st[2], st[3]};
    p.v = {a.v, st[4], st[5]};
    p.dout = {a.dout, st[6], st[7]};
    p.cu = a.cu_seqlens; p.n_seqs = a.n_seqs; p.tokens = a.tokens;
    p.heads = a.heads; p.kv_heads = a.kv_heads; p.head_dim = a.head_dim;
    p.type = a.dtype; p.causal = a.is_causal; p.scale = a.scale;
    p.out = a.out; p.lse = a.lse; p.low = a.out_low; p.zero_rest = a.zero_rest;
    p.out_in = a.out; p.lse_in = a.lse;
    p.dq = a.dq; p.dk = a.dk; p.dv = a.dv;
    p.ws = a.workspace; p.ws_bytes = a.ws_bytes > 0 ? (size_t)a.ws_bytes : 0;
    return p;
}

Pages pages(void* p, const long long* s) { return {p, s[1], s[2], s[3], s[0]}; }

}  // namespace

RAC_API long long rac_attention_packed_workspace(long long tokens, int n_seqs, int heads, int kv_heads, int head_dim,
                                                 int dtype, int backward) {
    if (tokens <= 0 || n_seqs < 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 0;
    return (long long)attention_packed_workspace(tokens, n_seqs, heads, kv_heads, head_dim, dtype, backward);
}

RAC_API int rac_attention_packed_async(const rac_attention_packed_args* args, void* stream) {
    if (!args) return record(kErrNullPtr, "rac_attention_packed_async");
    return record(attention_packed(packed(*args), static_cast<cudaStream_t>(stream)), "rac_attention_packed_async");
}

RAC_API int rac_attention_packed_backward_async(const rac_attention_packed_args* args, void* stream) {
    if (!args) return record(kErrNullPtr, "rac_attention_packed_backward_async");
    return record(attention_packed_backward(packed(*args), static_cast<cudaStream_t>(stream)),
                  "rac_attention_packed_backward_async");
}

RAC_API long long rac_attention_cached_workspace(int batch, int nodes, int heads, int kv_heads, int head_dim) {
    if (batch <= 0 || nodes <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 0;
    return (long long)attention_cached_workspace(batch, nodes, heads, kv_heads, head_dim);
}

RAC_API int rac_attention_cached_async(const rac_attention_cached_args* args, void* stream) {
    if (!args) return record(kErrNullPtr, "rac_attention_cached_async");
    const rac_attention_cached_args& a = *args;
    const long long* st = a.strides;
    CachedParams p{};
    p.q = a.q; p.q_batch = st[0]; p.q_node = st[1]; p.q_head = st[2];
    p.k = {const_cast<void*>(a.k_pages), st[3], st[4], st[5], 0};
    p.v = {const_cast<void*>(a.v_pages), st[6], st[7], st[8], 0};
    p.table = a.page_table; p.table_width = a.table_width; p.pages = a.n_pages; p.page_size = a.page_size;
    p.lengths = a.lengths; p.counts = a.counts; p.tree = a.tree;
    p.batch = a.batch; p.nodes = a.nodes; p.heads = a.heads; p.kv_heads = a.kv_heads; p.head_dim = a.head_dim;
    p.type = a.dtype; p.scale = a.scale; p.out = a.out; p.zero_rest = a.zero_rest;
    p.ws = a.workspace; p.ws_bytes = a.ws_bytes > 0 ? (size_t)a.ws_bytes : 0;
    return record(attention_cached(p, static_cast<cudaStream_t>(stream)), "rac_attention_cached_async");
}

RAC_API int rac_cache_append_async(const rac_cache_args* args, void* stream) {
    if (!args) return record(kErrNullPtr, "rac_cache_append_async");
    const rac_cache_args& a = *args;
    AppendParams p{};
    p.k = pages(a.k_pages, a.strides); p.v = pages(a.v_pages, a.strides + 4);
    p.nk = {a.k, a.strides[8], a.strides[9]}; p.nv = {a.v, a.strides[10], a.strides[11]};
    p.table = a.page_table; p.table_width = a.table_width; p.pages = a.n_pages; p.page_size = a.page_size;
    p.starts = a.starts; p.cu = a.cu_seqlens; p.batch = a.batch; p.tokens = a.tokens;
    p.kv_heads = a.kv_heads; p.head_dim = a.head_dim; p.type = a.dtype;
    return record(cache_append(p, static_cast<cudaStream_t>(stream)), "rac_cache_append_async");
}

RAC_API int rac_cache_copy_pages_async(const rac_cache_args* args, void* stream) {
    if (!args) return record(kErrNullPtr, "rac_cache_copy_pages_async");
    const rac_cache_args& a = *args;
    CopyPagesParams p{};
    p.k = pages(a.k_pages, a.strides); p.v = pages(a.v_pages, a.strides + 4);
    p.src = a.src; p.dst = a.dst; p.n = a.n; p.layers = a.layers; p.pages = a.n_pages; p.page_size = a.page_size;
    p.kv_heads = a.kv_heads; p.head_dim = a.head_dim; p.type = a.dtype;
    return record(cache_copy_pages(p, static_cast<cudaStream_t>(stream)), "rac_cache_copy_pages_async");
}

RAC_API int rac_cache_compact_async(const rac_cache_args* args, void* stream) {
    if (!args) return record(kErrNullPtr, "rac_cache_compact_async");
    const rac_cache_args& a = *args;
    CompactParams p{};
    p.k = pages(a.k_pages, a.strides); p.v = pages(a.v_pages, a.strides + 4);
    p.table = a.page_table; p.table_width = a.table_width; p.pages = a.n_pages; p.page_size = a.page_size;
    p.starts = a.starts; p.accepted = a.accepted; p.n_accepted = a.n_accepted; p.batch = a.batch; p.nodes = a.n;
    p.layers = a.layers; p.kv_heads = a.kv_heads; p.head_dim = a.head_dim; p.type = a.dtype;
    return record(cache_compact(p, static_cast<cudaStream_t>(stream)), "rac_cache_compact_async");
}
