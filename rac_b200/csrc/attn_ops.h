// attn_ops.h -- internal launchers of the packed-prompt and paged-cache
// attention and of the cache's page operations.  All take device pointers,
// enqueue on `s`, never synchronise and return a racb::Status.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace racb {

enum ElemType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };
inline int elem_bytes(int t) { return t == kF32 ? 4 : 2; }

// Rows (tokens) of heads: element (row, head, d) at p + row * row_stride + head * head_stride + d.
struct Rows {
    const void* p;
    long long row, head;
};

struct PackedParams {
    Rows q, k, v;
    const int* cu;
    int n_seqs;
    long long tokens;
    int heads, kv_heads, head_dim, type, causal;
    float scale;
    void* out;            // [tokens, heads, head_dim]
    float* lse;           // [heads, tokens], natural log; may be null forward
    void* low;            // like out: what rounding took from each sequence's first 128 rows; may be null
    int zero_rest;        // write zeros to the rows behind the last sequence
    // backward
    Rows dout;
    const void* out_in;   // the forward's output and lse
    const float* lse_in;
    void *dq, *dk, *dv;   // contiguous
    void* ws;
    size_t ws_bytes;
};

size_t attention_packed_workspace(long long tokens, int n_seqs, int heads, int kv_heads, int head_dim, int type,
                                  int backward);
// float16 and bfloat16, arguments checked.
int attention_packed_tc(const PackedParams& p, cudaStream_t s);
int attention_packed_backward_tc(const PackedParams& p, cudaStream_t s);
// float32, arguments checked.
size_t attention_packed_f32_workspace(long long tokens, int n_seqs, int heads, int kv_heads, int head_dim, int backward);
int attention_packed_f32(const PackedParams& p, int backward, cudaStream_t s);
bool rows_map(CUtensorMap* m, const Rows& r, int type, long long tokens, int heads, int hd);
int attention_packed(const PackedParams& p, cudaStream_t s);
int attention_packed_backward(const PackedParams& p, cudaStream_t s);

// Pages: element (page, head, slot, d) at p + page * page_stride + head * head_stride + slot * row_stride + d.
struct Pages {
    void* p;
    long long page, head, row, layer;
};

struct CachedParams {
    const void* q;        // [batch, nodes, heads, head_dim], strides below (elements)
    long long q_batch, q_node, q_head;
    Pages k, v;
    const int* table;     // [batch, table_width]
    int table_width;
    int pages, page_size;
    const int* lengths;   // [batch] rows in the cache, the new ones included
    const int* counts;    // [batch] new rows of each sequence, or null: nodes
    const long long* tree;  // [batch, nodes] bit masks over the new rows, or null: a chain
    int batch, nodes, heads, kv_heads, head_dim, type;
    float scale;
    void* out;            // [batch, nodes, heads, head_dim] contiguous
    int zero_rest;        // write zeros to the rows from counts[b] on
    void* ws;
    size_t ws_bytes;
};

size_t attention_cached_workspace(int batch, int nodes, int heads, int kv_heads, int head_dim);
// float16 and bfloat16 on `blocks` blocks, arguments checked.
size_t attention_cached_tc_workspace(int blocks, int nodes, int heads, int kv_heads, int head_dim);
int attention_cached_tc(const CachedParams& p, int blocks, cudaStream_t s);
int attention_cached(const CachedParams& p, cudaStream_t s);

struct AppendParams {
    Pages k, v;
    Rows nk, nv;          // the new rows
    const int* table;
    int table_width, pages, page_size;
    const int* starts;    // [batch] cache row of each sequence's first new row
    const int* cu;        // [batch + 1]
    int batch;
    long long tokens;
    int kv_heads, head_dim, type;
};
int cache_append(const AppendParams& p, cudaStream_t s);

struct CopyPagesParams {
    Pages k, v;
    const int *src, *dst;
    int n, layers, pages, page_size, kv_heads, head_dim, type;
};
int cache_copy_pages(const CopyPagesParams& p, cudaStream_t s);

struct CompactParams {
    Pages k, v;
    const int* table;
    int table_width, pages, page_size;
    const int* starts;     // [batch] cache row of node 0
    const int* accepted;   // [batch, nodes]
    const int* n_accepted; // [batch]
    int batch, nodes, layers, kv_heads, head_dim, type;
};
int cache_compact(const CompactParams& p, cudaStream_t s);

}  // namespace racb
