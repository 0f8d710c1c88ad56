// attention_packed.cu -- attention over packed prompts, forward and backward.
//
// Sequences of different lengths lie end to end in [tokens, heads, head_dim];
// query head h reads key/value head h / (heads / kv_heads).  Within a sequence
//   s_ij = scale q_i . k_j,  j <= i when causal,  p_ij = exp(s_ij - lse_i),
//   lse_i = log sum_j exp(s_ij),  o_i = sum_j p_ij v_j,
// and with do the output's gradient, D_i = do_i . o_i, ds_ij = p_ij (do_i . v_j - D_i):
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_{h,i} ds_ij q_i,  dv_j = sum_{h,i} p_ij do_i
// (sums over the query heads h that share the key/value head).  Every sum is
// held in 32 bits, in a fixed order: no atomics, the same bits every time.
#include "attn_common.cuh"

namespace racb {
namespace {

constexpr int kB = 64;            // query rows and keys of a tile
constexpr int kThreads = 128;     // thread (rg, cg): rows rg + 16 i (i < 4), columns cg + 8 j
constexpr int kPad = 4;           // floats behind a row: rows start in distinct bank groups

template <int HD>
constexpr int ld() { return HD + kPad; }

// Rows [row0, row0 + 64) of one head into a tile, zeros from `len` on.
template <typename T, int HD>
__device__ __forceinline__ void load_tile(float* dst, const T* __restrict__ src, long long row_stride, int row0,
                                          int len) {
    for (int e = threadIdx.x; e < kB * (HD / 4); e += kThreads) {
        const int r = e / (HD / 4), c = (e % (HD / 4)) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row0 + r < len) x = load4(src + (long long)(row0 + r) * row_stride + c);
        *reinterpret_cast<float4*>(dst + r * ld<HD>() + c) = x;
    }
}

// acc[i][j] = a_row . b_row over HD.
template <int HD>
__device__ __forceinline__ void dot_tile(float (&acc)[4][8], const float* A, const float* B) {
    const int rg = threadIdx.x >> 3, cg = threadIdx.x & 7;
    float2 s[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s[i][j] = make_float2(0.f, 0.f);
#pragma unroll 2
    for (int d = 0; d < HD; d += 4) {
        float4 a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(A + (rg + 16 * i) * ld<HD>() + d);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float4 b = *reinterpret_cast<const float4*>(B + (cg + 8 * j) * ld<HD>() + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i][j] = __ffma2_rn(make_float2(a[i].x, a[i].y), make_float2(b.x, b.y), s[i][j]);
                s[i][j] = __ffma2_rn(make_float2(a[i].z, a[i].w), make_float2(b.z, b.w), s[i][j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = s[i][j].x + s[i][j].y;
}

constexpr int kPld = kB + 1;      // weights: both the row- and the column-wise reads spread over the banks

// o[i][g] += sum_s w(row rg + 16 i, s) * V[s][...]; TR reads the weights transposed.
template <int HD, bool TR>
__device__ __forceinline__ void add_weighted(float4 (&o)[4][HD / 32], const float* W, const float* V) {
    const int rg = threadIdx.x >> 3, cg = threadIdx.x & 7;
#pragma unroll 4
    for (int s = 0; s < kB; ++s) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = TR ? W[s * kPld + rg + 16 * i] : W[(rg + 16 * i) * kPld + s];
#pragma unroll
        for (int g = 0; g < HD / 32; ++g) {
            const float4 v = *reinterpret_cast<const float4*>(V + s * ld<HD>() + cg * 4 + 32 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[i][g].x = fmaf(w[i], v.x, o[i][g].x);
                o[i][g].y = fmaf(w[i], v.y, o[i][g].y);
                o[i][g].z = fmaf(w[i], v.z, o[i][g].z);
                o[i][g].w = fmaf(w[i], v.w, o[i][g].w);
            }
        }
    }
}

template <int HD>
__device__ __forceinline__ void zero_acc(float4 (&o)[4][HD / 32]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int g = 0; g < HD / 32; ++g) o[i][g] = make_float4(0.f, 0.f, 0.f, 0.f);
}

// Rows [row0, row0 + 64) of o, times f, to a contiguous [tokens, heads, HD] tensor.
template <typename T, int HD>
__device__ __forceinline__ void store_rows(const float4 (&o)[4][HD / 32], const float (&f)[4], T* dst, long long start,
                                           int row0, int len, int heads, int head) {
    const int rg = threadIdx.x >> 3, cg = threadIdx.x & 7;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = row0 + rg + 16 * i;
        if (r >= len) continue;
        T* row = dst + ((start + r) * heads + head) * HD;
#pragma unroll
        for (int g = 0; g < HD / 32; ++g)
            store4(row + cg * 4 + 32 * g,
                   make_float4(o[i][g].x * f[i], o[i][g].y * f[i], o[i][g].z * f[i], o[i][g].w * f[i]));
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) k_packed_fwd(const PackedParams p) {
    extern __shared__ __align__(16) float smem[];
    float* Qs = smem;
    float* Ks = Qs + kB * ld<HD>();
    float* Vs = Ks + kB * ld<HD>();
    float* Ws = Vs + kB * ld<HD>();
    const PackedTile t = packed_tile(p.cu, p.n_seqs, p.tokens, kB, (long long)gridDim.x - 1 - blockIdx.x);
    if (t.row0 >= t.len) return;
    const int head = blockIdx.y, kvh = head / (p.heads / p.kv_heads);
    T* out = static_cast<T*>(p.out);
    float4 o[4][HD / 32];
    zero_acc<HD>(o);
    float m[4], l[4], inv[4] = {0.f, 0.f, 0.f, 0.f};
    if (t.seq == p.n_seqs) {                  // behind the last sequence
        if (p.zero_rest) store_rows<T, HD>(o, inv, out, t.start, t.row0, t.len, p.heads, head);
        return;
    }
    const T* q = static_cast<const T*>(p.q.p) + t.start * p.q.row + head * p.q.head;
    const T* k = static_cast<const T*>(p.k.p) + t.start * p.k.row + kvh * p.k.head;
    const T* v = static_cast<const T*>(p.v.p) + t.start * p.v.row + kvh * p.v.head;
    const int rg = threadIdx.x >> 3, cg = threadIdx.x & 7;
#pragma unroll
    for (int i = 0; i < 4; ++i) { m[i] = -INFINITY; l[i] = 0.f; }
    load_tile<T, HD>(Qs, q, p.q.row, t.row0, t.len);
    const int last = p.causal ? min(t.row0 + kB, t.len) : t.len;
    for (int k0 = 0; k0 < last; k0 += kB) {
        __syncthreads();
        load_tile<T, HD>(Ks, k, p.k.row, k0, t.len);
        load_tile<T, HD>(Vs, v, p.v.row, k0, t.len);
        __syncthreads();
        float s[4][8];
        dot_tile<HD>(s, Qs, Ks);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = t.row0 + rg + 16 * i;
            float mx = m[i];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = k0 + cg + 8 * j;
                s[i][j] = key < t.len && (!p.causal || key <= row) ? s[i][j] * p.scale : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            const float ref = mx == -INFINITY ? 0.f : mx;
            const float a = expf(m[i] - ref);
            m[i] = mx;
            l[i] *= a;
#pragma unroll
            for (int g = 0; g < HD / 32; ++g) { o[i][g].x *= a; o[i][g].y *= a; o[i][g].z *= a; o[i][g].w *= a; }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float e = expf(s[i][j] - ref);
                l[i] += e;
                Ws[(rg + 16 * i) * kPld + cg + 8 * j] = e;
            }
        }
        __syncthreads();
        add_weighted<HD, false>(o, Ws, Vs);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], off);
        inv[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
        const int row = t.row0 + rg + 16 * i;
        if (p.lse && cg == 0 && row < t.len)
            p.lse[(long long)head * p.tokens + t.start + row] = l[i] == 0.f ? -INFINITY : m[i] + logf(l[i]);
    }
    store_rows<T, HD>(o, inv, out, t.start, t.row0, t.len, p.heads, head);
}

// D = do . o: one warp per (token, head).
template <typename T, int HD>
__global__ void __launch_bounds__(256) k_packed_delta(const PackedParams p) {
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (w >= p.tokens * p.heads) return;
    const long long tok = w / p.heads;
    const int head = (int)(w % p.heads);
    const T* g = static_cast<const T*>(p.dout.p) + tok * p.dout.row + head * p.dout.head;
    const T* o = static_cast<const T*>(p.out_in) + w * HD;
    float s = 0.f;
    for (int c = lane * 4; c < HD; c += 128) {
        const float4 a = load4(g + c), b = load4(o + c);
        s += a.x * b.x + a.y * b.y + a.z * b.z + a.w * b.w;
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (lane == 0) static_cast<float*>(p.ws)[head * p.tokens + tok] = s;
}

// Weights p and ds of a 64 x 64 tile (rows: queries) from S and dP.
__device__ __forceinline__ void grad_weights(const PackedParams& p, const PackedTile& t, int head, int q0, int k0,
                                             float (&s)[4][8], float (&dp)[4][8]) {
    const int rg = threadIdx.x >> 3, cg = threadIdx.x & 7;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = q0 + rg + 16 * i;
        float lse = INFINITY, delta = 0.f;
        if (row < t.len) {
            lse = p.lse_in[(long long)head * p.tokens + t.start + row];
            delta = static_cast<float*>(p.ws)[(long long)head * p.tokens + t.start + row];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = k0 + cg + 8 * j;
            const bool seen = row < t.len && key < t.len && (!p.causal || key <= row) && lse != -INFINITY;
            const float w = seen ? expf(s[i][j] * p.scale - lse) : 0.f;
            s[i][j] = w;
            dp[i][j] = seen ? w * (dp[i][j] - delta) : 0.f;
        }
    }
}

__device__ __forceinline__ void put_weights(float* W, const float (&w)[4][8]) {
    const int rg = threadIdx.x >> 3, cg = threadIdx.x & 7;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) W[(rg + 16 * i) * kPld + cg + 8 * j] = w[i][j];
}

// dq of a tile of 64 queries.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) k_packed_dq(const PackedParams p) {
    extern __shared__ __align__(16) float smem[];
    float* Qs = smem;
    float* Gs = Qs + kB * ld<HD>();
    float* Ks = Gs + kB * ld<HD>();
    float* Vs = Ks + kB * ld<HD>();
    float* Ws = Vs + kB * ld<HD>();
    const PackedTile t = packed_tile(p.cu, p.n_seqs, p.tokens, kB, (long long)gridDim.x - 1 - blockIdx.x);
    if (t.row0 >= t.len) return;
    const int head = blockIdx.y, kvh = head / (p.heads / p.kv_heads);
    float4 o[4][HD / 32];
    zero_acc<HD>(o);
    const float f[4] = {p.scale, p.scale, p.scale, p.scale};
    T* dq = static_cast<T*>(p.dq);
    if (t.seq == p.n_seqs) {
        const float z[4] = {0.f, 0.f, 0.f, 0.f};
        store_rows<T, HD>(o, z, dq, t.start, t.row0, t.len, p.heads, head);
        return;
    }
    const T* q = static_cast<const T*>(p.q.p) + t.start * p.q.row + head * p.q.head;
    const T* g = static_cast<const T*>(p.dout.p) + t.start * p.dout.row + head * p.dout.head;
    const T* k = static_cast<const T*>(p.k.p) + t.start * p.k.row + kvh * p.k.head;
    const T* v = static_cast<const T*>(p.v.p) + t.start * p.v.row + kvh * p.v.head;
    load_tile<T, HD>(Qs, q, p.q.row, t.row0, t.len);
    load_tile<T, HD>(Gs, g, p.dout.row, t.row0, t.len);
    const int last = p.causal ? min(t.row0 + kB, t.len) : t.len;
    for (int k0 = 0; k0 < last; k0 += kB) {
        __syncthreads();
        load_tile<T, HD>(Ks, k, p.k.row, k0, t.len);
        load_tile<T, HD>(Vs, v, p.v.row, k0, t.len);
        __syncthreads();
        float s[4][8], dp[4][8];
        dot_tile<HD>(s, Qs, Ks);
        dot_tile<HD>(dp, Gs, Vs);
        grad_weights(p, t, head, t.row0, k0, s, dp);
        put_weights(Ws, dp);
        __syncthreads();
        add_weighted<HD, false>(o, Ws, Ks);
    }
    store_rows<T, HD>(o, f, dq, t.start, t.row0, t.len, p.heads, head);
}

// dk and dv of a tile of 64 keys, over all query heads of its group.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads) k_packed_dkv(const PackedParams p) {
    extern __shared__ __align__(16) float smem[];
    float* Qs = smem;
    float* Gs = Qs + kB * ld<HD>();
    float* Ks = Gs + kB * ld<HD>();
    float* Vs = Ks + kB * ld<HD>();
    float* Ws = Vs + kB * ld<HD>();
    float* Ds = Ws + kB * kPld;
    const PackedTile t = packed_tile(p.cu, p.n_seqs, p.tokens, kB, blockIdx.x);
    if (t.row0 >= t.len) return;
    const int kvh = blockIdx.y, group = p.heads / p.kv_heads;
    float4 dk[4][HD / 32], dv[4][HD / 32];
    zero_acc<HD>(dk);
    zero_acc<HD>(dv);
    const float f[4] = {p.scale, p.scale, p.scale, p.scale}, one[4] = {1.f, 1.f, 1.f, 1.f};
    if (t.seq < p.n_seqs) {
        const T* k = static_cast<const T*>(p.k.p) + t.start * p.k.row + kvh * p.k.head;
        const T* v = static_cast<const T*>(p.v.p) + t.start * p.v.row + kvh * p.v.head;
        load_tile<T, HD>(Ks, k, p.k.row, t.row0, t.len);
        load_tile<T, HD>(Vs, v, p.v.row, t.row0, t.len);
        for (int head = kvh * group; head < (kvh + 1) * group; ++head) {
            const T* q = static_cast<const T*>(p.q.p) + t.start * p.q.row + head * p.q.head;
            const T* g = static_cast<const T*>(p.dout.p) + t.start * p.dout.row + head * p.dout.head;
            for (int q0 = p.causal ? t.row0 : 0; q0 < t.len; q0 += kB) {
                __syncthreads();
                load_tile<T, HD>(Qs, q, p.q.row, q0, t.len);
                load_tile<T, HD>(Gs, g, p.dout.row, q0, t.len);
                __syncthreads();
                float s[4][8], dp[4][8];
                dot_tile<HD>(s, Qs, Ks);
                dot_tile<HD>(dp, Gs, Vs);
                grad_weights(p, t, head, q0, t.row0, s, dp);
                put_weights(Ws, s);
                put_weights(Ds, dp);
                __syncthreads();
                add_weighted<HD, true>(dv, Ws, Gs);
                add_weighted<HD, true>(dk, Ds, Qs);
            }
        }
    }
    store_rows<T, HD>(dk, f, static_cast<T*>(p.dk), t.start, t.row0, t.len, p.kv_heads, kvh);
    store_rows<T, HD>(dv, one, static_cast<T*>(p.dv), t.start, t.row0, t.len, p.kv_heads, kvh);
}

int launched() { return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda; }

template <typename T, int HD>
struct Fwd {
    static int run(const PackedParams& p, cudaStream_t s) {
        const size_t smem = sizeof(float) * (3 * kB * ld<HD>() + kB * kPld);
        if (cudaFuncSetAttribute(k_packed_fwd<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
            return kErrCuda;
        k_packed_fwd<T, HD><<<dim3((unsigned)packed_slots(p.tokens, p.n_seqs, kB), p.heads), kThreads, smem, s>>>(p);
        return launched();
    }
};

template <typename T, int HD>
struct Bwd {
    static int run(const PackedParams& p, cudaStream_t s) {
        k_packed_delta<T, HD><<<(unsigned)((p.tokens * p.heads + 7) / 8), 256, 0, s>>>(p);
        if (int st = launched()) return st;
        const unsigned slots = (unsigned)packed_slots(p.tokens, p.n_seqs, kB);
        const size_t sq = sizeof(float) * (4 * kB * ld<HD>() + kB * kPld), skv = sq + sizeof(float) * kB * kPld;
        if (cudaFuncSetAttribute(k_packed_dq<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sq) != cudaSuccess ||
            cudaFuncSetAttribute(k_packed_dkv<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)skv) != cudaSuccess)
            return kErrCuda;
        k_packed_dq<T, HD><<<dim3(slots, p.heads), kThreads, sq, s>>>(p);
        if (int st = launched()) return st;
        k_packed_dkv<T, HD><<<dim3(slots, p.kv_heads), kThreads, skv, s>>>(p);
        return launched();
    }
};

template <template <typename, int> class F, typename T>
int by_dim(const PackedParams& p, cudaStream_t s) {
    switch (p.head_dim) {
        case 32: return F<T, 32>::run(p, s);
        case 64: return F<T, 64>::run(p, s);
        case 128: return F<T, 128>::run(p, s);
        default: return kErrUnsupported;
    }
}

template <template <typename, int> class F>
int by_type(const PackedParams& p, cudaStream_t s) {
    switch (p.type) {
        case kF32: return by_dim<F, float>(p, s);
        case kF16: return by_dim<F, __half>(p, s);
        case kBF16: return by_dim<F, __nv_bfloat16>(p, s);
        default: return kErrUnsupported;
    }
}

// 16-byte loads: aligned base, strides of whole 16-byte units.
bool rows_ok(const Rows& r, int type) {
    const int e = elem_bytes(type);
    return (reinterpret_cast<uintptr_t>(r.p) & 15u) == 0 && (r.row * e) % 16 == 0 && (r.head * e) % 16 == 0 && r.row >= 0 && r.head >= 0;
}

int check(const PackedParams& p) {
    if (p.tokens < 0 || p.n_seqs < 0 || p.heads <= 0 || p.kv_heads <= 0 || p.heads % p.kv_heads) return kErrInvalidDim;
    if (p.type < kF32 || p.type > kBF16) return kErrUnsupported;
    if (p.head_dim != 32 && p.head_dim != 64 && p.head_dim != 128) return kErrUnsupported;
    if (p.tokens >= (1LL << 30) || p.heads > 65535 || p.n_seqs >= (1 << 30) ||
        packed_slots(p.tokens, p.n_seqs, kB) * p.heads >= (1LL << 31))
        return kErrInvalidDim;
    if (p.tokens && (!p.q.p || !p.k.p || !p.v.p || (p.n_seqs && !p.cu))) return kErrNullPtr;
    if (!rows_ok(p.q, p.type) || !rows_ok(p.k, p.type) || !rows_ok(p.v, p.type)) return kErrUnsupported;
    return kOk;
}

}  // namespace

// Backward: D, [heads, tokens], and two largest values.
size_t attention_packed_workspace(long long tokens, int, int heads, int, int, int, int backward) {
    return backward ? sizeof(float) * ((size_t)tokens * heads + 2) : 0;
}

int attention_packed(const PackedParams& p, cudaStream_t s) {
    if (int st = check(p)) return st;
    if (p.tokens == 0) return kOk;
    if (!p.out) return kErrNullPtr;
    if (reinterpret_cast<uintptr_t>(p.out) & 15u) return kErrUnsupported;
    if (p.type != kF32) return attention_packed_tc(p, s);
    return by_type<Fwd>(p, s);
}

int attention_packed_backward(const PackedParams& p, cudaStream_t s) {
    if (int st = check(p)) return st;
    if (p.tokens == 0) return kOk;
    if (!p.dout.p || !p.out_in || !p.lse_in || !p.dq || !p.dk || !p.dv) return kErrNullPtr;
    if (!rows_ok(p.dout, p.type)) return kErrUnsupported;
    if (!p.ws || p.ws_bytes < attention_packed_workspace(p.tokens, p.n_seqs, p.heads, p.kv_heads, p.head_dim, p.type, 1))
        return kErrAlloc;
    for (const void* x : {p.out_in, (const void*)p.dq, (const void*)p.dk, (const void*)p.dv})
        if (reinterpret_cast<uintptr_t>(x) & 15u) return kErrUnsupported;
    if (p.type != kF32) return attention_packed_backward_tc(p, s);
    return by_type<Bwd>(p, s);
}

}  // namespace racb
