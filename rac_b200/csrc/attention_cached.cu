// attention_cached.cu -- attention of new tokens over a paged key/value cache.
//
// Sequence b has lengths[b] rows in the cache; the last counts[b] of them are
// new, and queries (b, i, h), i < counts[b], attend over the rows before them
// (all visible) and over the new rows that their mask names: bit j of
// tree[b, i], or j <= i where there is no tree.  One token a sequence is the
// case nodes == 1.  o = sum_j p_j v_j, p = softmax(scale q . k_j) over the
// visible rows; a query that sees no row gives zeros.
#include "attn_common.cuh"

namespace racb {
namespace {

constexpr int kThreads = 128;

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) k_cached_simple(const CachedParams p, unsigned int* err) {
    __shared__ float qs[HD], w[kThreads], red[8];
    __shared__ long long koff[kThreads], voff[kThreads];
    const int head = blockIdx.x, node = blockIdx.y, b = blockIdx.z;
    const int kvh = head / (p.heads / p.kv_heads);
    const long long cap = (long long)p.table_width * p.page_size;
    const long long len = max(0LL, min((long long)p.lengths[b], cap));
    const int cnt = p.counts ? max(0, min(p.counts[b], p.nodes)) : p.nodes;
    T* out = static_cast<T*>(p.out) + (((long long)b * p.nodes + node) * p.heads + head) * HD;
    const int tid = threadIdx.x;
    if (node >= cnt) {
        if (p.zero_rest && tid < HD) out[tid] = from_f32<T>(0.f);
        return;
    }
    const long long prefix = max(0LL, len - cnt);
    const unsigned long long sees = p.tree ? (unsigned long long)p.tree[(long long)b * p.nodes + node]
                                           : ~0ull >> (63 - node);
    const T* q = static_cast<const T*>(p.q) + b * p.q_batch + node * p.q_node + head * p.q_head;
    if (tid < HD) qs[tid] = to_f32(q[tid]) * p.scale;
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (long long r0 = 0; r0 < len; r0 += kThreads) {
        __syncthreads();
        const long long r = r0 + tid;
        bool ok = r < len && (r < prefix || ((sees >> min(63LL, r - prefix)) & 1));
        if (ok) {
            const int pg = p.table[(long long)b * p.table_width + r / p.page_size];
            if (pg < 0 || pg >= p.pages) { ok = false; atomicOr(err, kErrBadPage); }
            koff[tid] = pg * p.k.page + kvh * p.k.head + (r % p.page_size) * p.k.row;
            voff[tid] = pg * p.v.page + kvh * p.v.head + (r % p.page_size) * p.v.row;
        }
        float s = -INFINITY;
        if (ok) {
            const T* k = static_cast<const T*>(p.k.p) + koff[tid];
            s = 0.f;
            for (int c = 0; c < HD; c += 4) {
                const float4 x = load4(k + c);
                s += qs[c] * x.x + qs[c + 1] * x.y + qs[c + 2] * x.z + qs[c + 3] * x.w;
            }
        } else {
            koff[tid] = voff[tid] = -1;
        }
        float mx = s;
        for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        if ((tid & 31) == 0) red[tid >> 5] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        mx = fmaxf(mx, m);
        const float ref = mx == -INFINITY ? 0.f : mx, a = expf(m - ref);
        m = mx;
        w[tid] = ok ? expf(s - ref) : 0.f;
        __syncthreads();
        l *= a;
        o *= a;
        for (int i = 0; i < kThreads; ++i) {
            l += w[i];
            if (tid < HD && voff[i] >= 0) o += w[i] * to_f32(static_cast<const T*>(p.v.p)[voff[i] + tid]);
        }
    }
    if (tid < HD) out[tid] = from_f32<T>(l == 0.f ? 0.f : o / l);
}

template <typename T>
int by_dim(const CachedParams& p, unsigned int* err, cudaStream_t s) {
    const dim3 grid(p.heads, p.nodes, p.batch);
    switch (p.head_dim) {
        case 32: k_cached_simple<T, 32><<<grid, kThreads, 0, s>>>(p, err); break;
        case 64: k_cached_simple<T, 64><<<grid, kThreads, 0, s>>>(p, err); break;
        case 128: k_cached_simple<T, 128><<<grid, kThreads, 0, s>>>(p, err); break;
        default: return kErrUnsupported;
    }
    return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

}  // namespace

// Blocks of the tensor-core kernel: one an SM.
static int block_count() {
    static int per_dev[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return 0; }
    if (per_dev[dev] == 0) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) { cudaGetLastError(); return 0; }
        per_dev[dev] = n;
    }
    return per_dev[dev];
}

size_t attention_cached_workspace(int, int nodes, int heads, int kv_heads, int head_dim) {
    return attention_cached_tc_workspace(block_count(), nodes, heads, kv_heads, head_dim);
}

int attention_cached(const CachedParams& p, cudaStream_t s) {
    if (p.batch < 0 || p.nodes < 0 || p.heads <= 0 || p.kv_heads <= 0 || p.heads % p.kv_heads || p.nodes > 64 ||
        p.table_width < 0 || p.pages < 0 || p.page_size <= 0 || p.batch > 65535)
        return kErrInvalidDim;
    if (p.head_dim != 32 && p.head_dim != 64 && p.head_dim != 128) return kErrUnsupported;
    if (p.type < kF32 || p.type > kBF16) return kErrUnsupported;
    if (p.batch == 0 || p.nodes == 0) return kOk;
    if (!p.q || !p.lengths || !p.out || (p.pages && (!p.k.p || !p.v.p)) || (p.table_width && !p.table)) return kErrNullPtr;
    const int e = elem_bytes(p.type);
    for (long long st : {p.q_batch, p.q_node, p.q_head, p.k.page, p.k.head, p.k.row, p.v.page, p.v.head, p.v.row})
        if (st * e % 16) return kErrUnsupported;
    for (const void* x : {p.q, (const void*)p.k.p, (const void*)p.v.p, (const void*)p.out})
        if (reinterpret_cast<uintptr_t>(x) & 15u) return kErrUnsupported;
    if ((long long)p.batch * p.kv_heads * ((long long)p.nodes * (p.heads / p.kv_heads)) >= (1LL << 31)) return kErrInvalidDim;
    if (p.type != kF32) {
        const int blocks = block_count();
        if (blocks == 0) return kErrCuda;
        if (!p.ws || p.ws_bytes < attention_cached_tc_workspace(blocks, p.nodes, p.heads, p.kv_heads, p.head_dim))
            return kErrAlloc;
        return attention_cached_tc(p, blocks, s);
    }
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return kErrCuda; }
    unsigned int* err = device_error_word(dev);
    if (!err) return kErrCuda;
    switch (p.type) {
        case kF32: return by_dim<float>(p, err, s);
        default: return kErrUnsupported;
    }
}

}  // namespace racb
