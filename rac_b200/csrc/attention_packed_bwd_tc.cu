// attention_packed_bwd_tc.cu -- gradients of attention over packed prompts on
// the tensor cores, float16 and bfloat16.
//
// Two kinds of block, each with its sums in tensor memory and no atomics: one keeps a
// tile of 128 queries and runs over the keys (dq), one keeps a tile of 128 keys
// and runs over the queries of all heads of its group (dk and dv).  Both
// compute S and dP anew: seven products where one kernel would do with five,
// but dq would then be added up by atomics, in an order that changes.
//
// In the dk/dv blocks everything is transposed, so that P^T and dS^T have a key
// a lane and feed dV += P^T dO and dK += dS^T Q from tensor memory.  The order
//   dV(i), S(i+1), dK(i), dP(i+1), dV(i+1), ...
// keeps the tensor core at work while the weights P(i+1) are taken from S(i+1)
// and dS(i+1) from dP(i+1): P(i) lies in S(i)'s columns and dS(i) in dP(i)'s, so
// that four 128-column blocks (S, dP, dK, dV) fill the 512 columns.
//
// float16: weights below 2^-14 and dS of small gradients would fall among the
// subnormal numbers and lose their digits.  P carries a factor 2^10, and dS a
// power of two that keeps it below the type's largest value, taken from the largest
// |do| and |v| of the sequence and key/value head: |dS| <= 2 head_dim max|do| max|v|.
// (Of all sequences together, one of large gradients took the digits of the others.)
//
// Bound: the seven products (the tensor pipe is busy half of the time) and the
// way of P and dS through registers between them.  8192 causal tokens in three
// sequences, 32 heads of 128 on 8, bf16, forward and backward: 1.11 ms, of which
// these kernels take 0.76 and D 0.03.
#include "attn_common.cuh"
#include "tensor_core.cuh"

namespace racb {
namespace {

using namespace tc;

constexpr int kTile = 128;
// Warps 0-3 and 4-7: columns 0-63 and 64-127 of a tile, a thread a row; 8: matrix
// instructions; 9: loads; 10: row statistics.
constexpr int kThreads = 384;
constexpr int kLaunchRegs = 168, kMathRegs = 216, kOtherRegs = 72;
static_assert(kMathRegs * 256 + kOtherRegs * 128 <= kLaunchRegs * kThreads, "register split");

struct BwdArgs {
    CUtensorMap q, k, v, g;
    const int* cu;
    int n_seqs, heads, kv_heads, group, causal;
    long long tokens;
    float c, scale;                        // scale * log2(e), scale
    const float *lse, *delta;              // [heads, tokens]
    const float* top;                      // float16: max |do|, max |v| of each sequence and key/value head
    void *dq, *dk, *dv;
    unsigned int* err;
};

// Power of two on dS of a sequence's key/value head, and exponent on P.
template <typename T>
__device__ __forceinline__ float ds_factor(const BwdArgs& a, int seq, int kvh, int hd) {
    if (!std::is_same<T, __half>::value) return 1.f;
    const float* top = a.top + 2 * ((long long)seq * a.kv_heads + kvh);
    const float b = 2.f * hd * top[0] * top[1];
    if (!(b > 0.f) || b > 1e30f) return 1.f;
    int e;
    frexpf(b, &e);                         // b <= 2^e
    return ldexpf(1.f, min(max(15 - e, -100), 100));
}
template <typename T> constexpr int p_shift() { return std::is_same<T, __half>::value ? 10 : 0; }

template <int HD>
struct Shape {
    static constexpr int SW = HD * 2 < 128 ? HD * 2 : 128;
    static constexpr int BOXES = HD * 2 / SW;
    static constexpr int BOX = kTile * SW;
    static constexpr int TILE = BOXES * BOX;
    static constexpr int A = 3, B = 2;     // ring of Q (dk/dv) or K (dq), ring of dO or V
    static constexpr int STAT = (2 + A + B) * TILE;
    static constexpr int BARS = STAT + 4 * kTile * 4;
    static constexpr int SMEM = BARS + 256;
};
static_assert(Shape<128>::SMEM <= 227 * 1024, "shared memory");

template <int HD>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* m, int head, int row, uint64_t* bar) {
    using Sh = Shape<HD>;
#pragma unroll
    for (int b = 0; b < Sh::BOXES; ++b) load_3d(dst + b * Sh::BOX, m, b * (Sh::SW / 2), head, row, bar);
}

// Rows [r0, 128) of a tile become zeros, by one warp.
template <int HD>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int r0) {
    using Sh = Shape<HD>;
    const int n = (kTile - r0) * (Sh::SW / 16), lane = threadIdx.x & 31;
    for (int e = lane; e < n * Sh::BOXES; e += 32)
        *reinterpret_cast<uint4*>(tile + (e / n) * Sh::BOX + r0 * Sh::SW + (e % n) * 16) = make_uint4(0, 0, 0, 0);
}

// D = A B^T over HD, both tiles row-major in shared memory.
template <typename T, int HD>
__device__ __forceinline__ void mma_rows(uint32_t d, const uint8_t* a, const uint8_t* b) {
    using Sh = Shape<HD>;
    product_ss<HD / 16, Sh::SW>(d, smem(a), smem(b), Sh::BOX, instruction<T>(kTile, kTile, false));
}
// D (+)= W B, W [128, 128] packed in tensor memory (columns 0-31 and 64-95 of its
// block), B's rows summed over.
template <typename T, int HD>
__device__ __forceinline__ void mma_weights(uint32_t d, uint32_t w, const uint8_t* b, bool add) {
    using Sh = Shape<HD>;
    constexpr uint32_t instr = instruction<T>(kTile, HD, true);
    const uint64_t db = operand<Sh::SW>(smem(b), Sh::BOX, 8 * Sh::SW);
#pragma unroll
    for (int k = 0; k < kTile; k += 16)
        mma_ts(d, w + (k < 64 ? k / 2 : 64 + (k - 64) / 2), db + (k * Sh::SW >> 4), instr, add || k > 0);
}

// A row of HD sums, times f, to global memory.
template <typename T, int HD>
__device__ __forceinline__ void store_row(uint32_t t, float f, T* dst, bool live, int b0 = 0, int step = 1) {
#pragma unroll
    for (int b = 0; b < HD / 32; ++b) {
        if (b % step != b0) continue;
        uint32_t o[32];
        ld32(o, t + 32 * b);
        wait_ld();
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            uint4 u;
            u.x = pack2<T>(__uint_as_float(o[i]) * f, __uint_as_float(o[i + 1]) * f);
            u.y = pack2<T>(__uint_as_float(o[i + 2]) * f, __uint_as_float(o[i + 3]) * f);
            u.z = pack2<T>(__uint_as_float(o[i + 4]) * f, __uint_as_float(o[i + 5]) * f);
            u.w = pack2<T>(__uint_as_float(o[i + 6]) * f, __uint_as_float(o[i + 7]) * f);
            *reinterpret_cast<uint4*>(dst + 32 * b + i) = u;
        }
    }
}

// Rows behind the last sequence: zeros.
template <typename T, int HD>
__device__ __forceinline__ void zero_out(T* dst, long long row, int row0, int len) {
    const int n = min(kTile, len - row0) * (HD / 8);
    for (int e = threadIdx.x; e < n; e += kThreads)
        *reinterpret_cast<uint4*>(dst + (row0 + e / (HD / 8)) * row + (e % (HD / 8)) * 8) = make_uint4(0, 0, 0, 0);
}

constexpr float kLog2e = 1.4426950408889634f;

// ── dk, dv ────────────────────────────────────────────────────────────────
template <typename T, int HD>
__device__ __forceinline__ void block_dkv(const BwdArgs& a, uint8_t* sm, unsigned block) {
    using Sh = Shape<HD>;
    constexpr int NA = Sh::A, NB = Sh::B;
    uint8_t *ks = sm, *vs = sm + Sh::TILE, *qr = sm + 2 * Sh::TILE, *gr = qr + NA * Sh::TILE;
    float* st_lse = reinterpret_cast<float*>(sm + Sh::STAT);       // negative; [2][128]
    float* st_d = st_lse + 2 * kTile;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Sh::BARS);
    uint64_t *kv_full = bars, *q_full = bars + 2, *q_empty = q_full + NA, *g_full = q_empty + NA, *g_empty = g_full + NB,
             *stat_full = g_empty + NB, *stat_empty = stat_full + 2, *s_ready = stat_empty + 2, *dp_ready = s_ready + 1,
             *p_ready = dp_ready + 1, *ds_ready = p_ready + 1, *done = ds_ready + 1, *fixed = done + 1;
    uint32_t* tmem_base = reinterpret_cast<uint32_t*>(fixed + NB);
    volatile int* gone = reinterpret_cast<volatile int*>(tmem_base + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int kvh = block % a.kv_heads;
    const PackedTile t = packed_tile(a.cu, a.n_seqs, a.tokens, kTile, block / a.kv_heads);
    if (t.row0 >= t.len) return;
    const long long out_row = (long long)a.kv_heads * HD;
    T* dk = static_cast<T*>(a.dk) + (t.start * a.kv_heads + kvh) * HD;
    T* dv = static_cast<T*>(a.dv) + (t.start * a.kv_heads + kvh) * HD;
    if (t.seq == a.n_seqs) {
        zero_out<T, HD>(dk, out_row, t.row0, t.len);
        zero_out<T, HD>(dv, out_row, t.row0, t.len);
        return;
    }
    const int first = a.causal ? t.row0 / kTile : 0;               // query tiles that see this one
    const int nq = (t.len + kTile - 1) / kTile - first;
    const int n = nq * a.group;
    const bool ragged = t.len % kTile != 0;                        // the last query tile of each head

    // The loading thread sets up the barriers and sends for the first tiles while
    // tensor memory is allocated: a block's first product waits for little else.
    if (threadIdx.x == 32 * 9) {
        *gone = 0;
        bar_init(kv_full, 1);
        bar_init(kv_full + 1, 1);
        for (int i = 0; i < NA; ++i) { bar_init(q_full + i, 1); bar_init(q_empty + i, 1); }
        for (int i = 0; i < NB; ++i) { bar_init(g_full + i, 1); bar_init(g_empty + i, 1); }
        for (int i = 0; i < 2; ++i) { bar_init(stat_full + i, 1); bar_init(stat_empty + i, 256); }
        bar_init(s_ready, 1); bar_init(dp_ready, 1); bar_init(p_ready, 256); bar_init(ds_ready, 256);
        bar_init(done, 1);
        for (int i = 0; i < NB; ++i) bar_init(fixed + i, 1);
        bar_init_done();
        const int k0 = (int)t.start + t.row0, q0 = (int)t.start + first * kTile;
        bar_expect(kv_full, Sh::TILE);
        load_tile<HD>(ks, &a.k, kvh, k0, kv_full);
        bar_expect(q_full, Sh::TILE);
        load_tile<HD>(qr, &a.q, kvh * a.group, q0, q_full);
        bar_expect(kv_full + 1, Sh::TILE);
        load_tile<HD>(vs, &a.v, kvh, k0, kv_full + 1);
        bar_expect(g_full, Sh::TILE);
        load_tile<HD>(gr, &a.g, kvh * a.group, q0, g_full);
    }
    if (warp == 8) tmem_alloc(tmem_base, 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm = *tmem_base, tS = tm, tP = tm + 128, tV = tm + 256, tK = tm + 384;

    if (warp >= 8) {
        fewer_registers<kOtherRegs>();
        if (warp == 9) {
            auto head_of = [&](int i) { return kvh * a.group + i / nq; };
            auto row_of = [&](int i) { return (int)t.start + (first + i % nq) * kTile; };
            bool ok = true;
            // Entry i is loaded as soon as its places are free; in a sequence's last
            // tile the rows behind it are cleared once they have landed: the weights
            // there are 0, and 0 times another sequence's NaN would not be.
            for (int i = 0; ok && i < n; ++i) {
                const int sa = i % NA, sb = i % NB;
                if (i >= NA) ok = bar_wait(q_empty + sa, (i / NA - 1) & 1, gone);
                if (ok && i >= NB) ok = bar_wait(g_empty + sb, (i / NB - 1) & 1, gone);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0 && i) {
                    bar_expect(q_full + sa, Sh::TILE);
                    load_tile<HD>(qr + sa * Sh::TILE, &a.q, head_of(i), row_of(i), q_full + sa);
                    bar_expect(g_full + sb, Sh::TILE);
                    load_tile<HD>(gr + sb * Sh::TILE, &a.g, head_of(i), row_of(i), g_full + sb);
                }
                __syncwarp();
                if (ragged && i % nq == nq - 1) {
                    ok = bar_wait(q_full + sa, (i / NA) & 1, gone) && bar_wait(g_full + sb, (i / NB) & 1, gone);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    zero_rows<HD>(qr + sa * Sh::TILE, t.len % kTile);
                    zero_rows<HD>(gr + sb * Sh::TILE, t.len % kTile);
                    fence_async_smem();
                    __syncwarp();
                }
                if (lane == 0) bar_arrive(fixed + sb);
            }
        } else if (warp == 8) {
            if (lane == 0) {
                auto ready = [&](int i) { return bar_wait(fixed + i % NB, (i / NB) & 1, gone); };
                bool ok = bar_wait(kv_full, 0, gone) && bar_wait(q_full, 0, gone) && ready(0);
                if (ok) {
                    mma_rows<T, HD>(tS, ks, qr);
                    commit(s_ready);
                    ok = bar_wait(kv_full + 1, 0, gone) && bar_wait(g_full, 0, gone);
                }
                if (ok) {
                    mma_rows<T, HD>(tP, vs, gr);
                    commit(dp_ready);
                }
                for (int i = 0; ok && i < n; ++i) {
                    const bool more = i + 1 < n;
                    const int sa = i % NA, sb = i % NB, na = (i + 1) % NA, nb = (i + 1) % NB;
                    ok = bar_wait(p_ready, i & 1, gone);
                    if (!ok) break;
                    fence_after();
                    mma_weights<T, HD>(tV, tS, gr + sb * Sh::TILE, i > 0);
                    commit(g_empty + sb);
                    if (more) {
                        ok = bar_wait(q_full + na, ((i + 1) / NA) & 1, gone) && ready(i + 1);
                        if (!ok) break;
                        mma_rows<T, HD>(tS, ks, qr + na * Sh::TILE);
                        commit(s_ready);
                    }
                    ok = bar_wait(ds_ready, i & 1, gone);
                    if (!ok) break;
                    fence_after();
                    mma_weights<T, HD>(tK, tP, qr + sa * Sh::TILE, i > 0);
                    commit(q_empty + sa);
                    if (more) {
                        ok = bar_wait(g_full + nb, ((i + 1) / NB) & 1, gone);
                        if (!ok) break;
                        mma_rows<T, HD>(tP, vs, gr + nb * Sh::TILE);
                        commit(dp_ready);
                    }
                }
                if (ok) commit(done);
            }
            __syncwarp();
        } else if (warp == 10) {
            // Row statistics of each query tile; a row behind the sequence has weight exp2(-inf).
            const float gf = ds_factor<T>(a, t.seq, kvh, HD) * (1.f / (1 << p_shift<T>()));
            for (int i = 0; i < n; ++i) {
                const int sl = i & 1;
                const bool ok = i < 2 || bar_wait(stat_empty + sl, (i / 2 - 1) & 1, gone);
                if (!__all_sync(0xffffffffu, ok)) break;
                const long long at = (long long)(kvh * a.group + i / nq) * a.tokens + t.start;
                for (int r = lane; r < kTile; r += 32) {
                    const int row = (first + i % nq) * kTile + r;
                    float x = INFINITY, d = 0.f;
                    if (row < t.len) {
                        x = a.lse[at + row];
                        x = x == -INFINITY ? INFINITY : x * kLog2e - p_shift<T>();
                        d = a.delta[at + row] * gf;
                    }
                    st_lse[sl * kTile + r] = -x;
                    st_d[sl * kTile + r] = -d;
                }
                __syncwarp();
                if (lane == 0) bar_arrive(stat_full + sl);
            }
        }
    } else {
        more_registers<kMathRegs>();
        const int half = warp >> 2, row = t.row0 + (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s0 = tS + lanes + 64 * half, p0 = tP + lanes + 64 * half;
        const float gf = ds_factor<T>(a, t.seq, kvh, HD) * (1.f / (1 << p_shift<T>()));
        bool ok = true;
        for (int i = 0; i < n; ++i) {
            const int sl = i & 1;
            ok = bar_wait(stat_full + sl, (i / 2) & 1, gone) && bar_wait(s_ready, i & 1, gone);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            const bool diag = a.causal && i % nq == 0;
            const int see = diag ? row - t.row0 - 64 * half : -1;          // columns from here on see this key
            const float* lse = st_lse + sl * kTile + 64 * half;
            const float* dd = st_d + sl * kTile + 64 * half;
            float2 p[32];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t s[32], w[16];
                ld32(s, s0 + 32 * b);
                wait_ld();
#pragma unroll
                for (int x = 0; x < 16; x += 2) {
                    const float4 m = *reinterpret_cast<const float4*>(lse + 32 * b + 2 * x);
                    p[16 * b + x] = exp2_both(__ffma2_rn(pair(s[2 * x], s[2 * x + 1]), both(a.c), make_float2(m.x, m.y)));
                    p[16 * b + x + 1] = exp2_both(__ffma2_rn(pair(s[2 * x + 2], s[2 * x + 3]), both(a.c), make_float2(m.z, m.w)));
                }
                if (diag) {
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        if (32 * b + 2 * x < see) p[16 * b + x].x = 0.f;
                        if (32 * b + 2 * x + 1 < see) p[16 * b + x].y = 0.f;
                    }
                }
#pragma unroll
                for (int x = 0; x < 16; ++x) w[x] = pack2<T>(p[16 * b + x].x, p[16 * b + x].y);
                st16(s0 + 16 * b, w);
            }
            wait_st();
            fence_before();
            bar_arrive(p_ready);
            ok = bar_wait(dp_ready, i & 1, gone);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t s[32], w[16];
                ld32(s, p0 + 32 * b);
                wait_ld();
#pragma unroll
                for (int x = 0; x < 16; x += 2) {
                    const float4 m = *reinterpret_cast<const float4*>(dd + 32 * b + 2 * x);
                    float2 e0 = __fmul2_rn(p[16 * b + x], __ffma2_rn(pair(s[2 * x], s[2 * x + 1]), both(gf), make_float2(m.x, m.y)));
                    float2 e1 = __fmul2_rn(p[16 * b + x + 1], __ffma2_rn(pair(s[2 * x + 2], s[2 * x + 3]), both(gf), make_float2(m.z, m.w)));
                    if (diag) {
                        if (32 * b + 2 * x < see) e0.x = 0.f;
                        if (32 * b + 2 * x + 1 < see) e0.y = 0.f;
                        if (32 * b + 2 * x + 2 < see) e1.x = 0.f;
                        if (32 * b + 2 * x + 3 < see) e1.y = 0.f;
                    }
                    w[x] = pack2<T>(e0.x, e0.y);
                    w[x + 1] = pack2<T>(e1.x, e1.y);
                }
                st16(p0 + 16 * b, w);
            }
            wait_st();
            fence_before();
            bar_arrive(ds_ready);
            bar_arrive(stat_empty + sl);
        }
        if (ok) ok = bar_wait(done, 0, gone);
        if (__all_sync(0xffffffffu, ok)) {
            fence_after();
            const bool live = row < t.len;
            if (half == 0) store_row<T, HD>(tV + lanes, 1.f / (1 << p_shift<T>()), dv + row * out_row, live);
            else store_row<T, HD>(tK + lanes, a.scale / ds_factor<T>(a, t.seq, kvh, HD), dk + row * out_row, live);
        }
    }
    fence_before();
    __syncthreads();
    settle(gone);
    fence_after();
    if (warp == 8) tmem_free(tm, 512);
    if (threadIdx.x == 0 && *gone) atomicOr(a.err, kErrTcWait);
}

// ── dq ────────────────────────────────────────────────────────────────────
// S has two blocks of columns, so that S(j+2) can follow dQ(j), whose weights
// dS(j) lie in S(j)'s; the order is dP(j+1), dQ(j), S(j+2).
template <typename T, int HD>
__device__ __forceinline__ void block_dq(const BwdArgs& a, uint8_t* sm, unsigned block, unsigned blocks) {
    using Sh = Shape<HD>;
    constexpr int NA = Sh::A, NB = Sh::B;
    uint8_t *qs = sm, *gs = sm + Sh::TILE, *kr = sm + 2 * Sh::TILE, *vr = kr + NA * Sh::TILE;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Sh::BARS);
    uint64_t *qg_full = bars, *k_full = bars + 2, *k_empty = k_full + NA, *v_full = k_empty + NA, *v_empty = v_full + NB,
             *s_ready = v_empty + NB, *dp_ready = s_ready + 2, *ds_ready = dp_ready + 1, *done = ds_ready + 1,
             *fixed = done + 1;
    uint32_t* tmem_base = reinterpret_cast<uint32_t*>(fixed + 1);
    volatile int* gone = reinterpret_cast<volatile int*>(tmem_base + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int head = block % a.heads, kvh = head / a.group;
    const PackedTile t = packed_tile(a.cu, a.n_seqs, a.tokens, kTile, (blocks - 1 - block) / a.heads);
    if (t.row0 >= t.len) return;
    const long long out_row = (long long)a.heads * HD;
    T* dq = static_cast<T*>(a.dq) + (t.start * a.heads + head) * HD;
    if (t.seq == a.n_seqs) {
        zero_out<T, HD>(dq, out_row, t.row0, t.len);
        return;
    }
    const int last = a.causal ? min(t.row0 + kTile, t.len) : t.len;
    const int n = (last + kTile - 1) / kTile;
    const bool ragged = n * kTile > t.len;

    if (threadIdx.x == 32 * 9) {
        *gone = 0;
        bar_init(qg_full, 1);
        bar_init(qg_full + 1, 1);
        for (int i = 0; i < NA; ++i) { bar_init(k_full + i, 1); bar_init(k_empty + i, 1); }
        for (int i = 0; i < NB; ++i) { bar_init(v_full + i, 1); bar_init(v_empty + i, 1); }
        bar_init(s_ready, 1); bar_init(s_ready + 1, 1); bar_init(dp_ready, 1); bar_init(ds_ready, 256);
        bar_init(done, 1); bar_init(fixed, 1);
        bar_init_done();
        const int r0 = (int)t.start;
        bar_expect(qg_full, Sh::TILE);
        load_tile<HD>(qs, &a.q, head, r0 + t.row0, qg_full);
        bar_expect(k_full, Sh::TILE);
        load_tile<HD>(kr, &a.k, kvh, r0, k_full);
        bar_expect(qg_full + 1, Sh::TILE);
        load_tile<HD>(gs, &a.g, head, r0 + t.row0, qg_full + 1);
        bar_expect(v_full, Sh::TILE);
        load_tile<HD>(vr, &a.v, kvh, r0, v_full);
    }
    if (warp == 8) tmem_alloc(tmem_base, 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm = *tmem_base, tS = tm, tP = tm + 256, tQ = tm + 384;

    if (warp >= 8) {
        fewer_registers<kOtherRegs>();
        if (warp == 9) {
            if (lane == 0) {
                const int r0 = (int)t.start;
                for (int j = 1; j < n; ++j) {
                    const int sa = j % NA, sb = j % NB;
                    if (j >= NA && !bar_wait(k_empty + sa, (j / NA - 1) & 1, gone)) break;
                    bar_expect(k_full + sa, Sh::TILE);
                    load_tile<HD>(kr + sa * Sh::TILE, &a.k, kvh, r0 + j * kTile, k_full + sa);
                    if (j >= NB && !bar_wait(v_empty + sb, (j / NB - 1) & 1, gone)) break;
                    bar_expect(v_full + sb, Sh::TILE);
                    load_tile<HD>(vr + sb * Sh::TILE, &a.v, kvh, r0 + j * kTile, v_full + sb);
                }
            }
            __syncwarp();
            if (ragged) {                   // keys behind the sequence: their dS is 0, 0 times NaN would not be
                const int j = n - 1;
                if (bar_wait(k_full + j % NA, (j / NA) & 1, gone)) {
                    zero_rows<HD>(kr + (j % NA) * Sh::TILE, t.len - j * kTile);
                    fence_async_smem();
                }
                __syncwarp();
                if (lane == 0) bar_arrive(fixed);
            }
        } else if (warp == 8) {
            if (lane == 0) {
                auto scores = [&](int j) {
                    if (!bar_wait(k_full + j % NA, (j / NA) & 1, gone)) return false;
                    if (ragged && j == n - 1 && !bar_wait(fixed, 0, gone)) return false;
                    mma_rows<T, HD>(tS + 128 * (j & 1), qs, kr + (j % NA) * Sh::TILE);
                    commit(s_ready + (j & 1));
                    return true;
                };
                auto dps = [&](int j) {
                    if (!bar_wait(v_full + j % NB, (j / NB) & 1, gone)) return false;
                    mma_rows<T, HD>(tP, gs, vr + (j % NB) * Sh::TILE);
                    commit(dp_ready);
                    commit(v_empty + j % NB);
                    return true;
                };
                bool ok = bar_wait(qg_full, 0, gone) && scores(0) && bar_wait(qg_full + 1, 0, gone) && dps(0);
                if (ok && n > 1) ok = scores(1);
                for (int j = 0; ok && j < n; ++j) {
                    ok = bar_wait(ds_ready, j & 1, gone);
                    if (!ok) break;
                    fence_after();
                    if (j + 1 < n) ok = dps(j + 1);
                    if (!ok) break;
                    mma_weights<T, HD>(tQ, tS + 128 * (j & 1), kr + (j % NA) * Sh::TILE, j > 0);
                    commit(k_empty + j % NA);
                    if (j + 2 < n) ok = scores(j + 2);
                }
                if (ok) commit(done);
            }
            __syncwarp();
        }
    } else {
        more_registers<kMathRegs>();
        const int half = warp >> 2, row = t.row0 + (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t p0 = tP + lanes + 64 * half;
        const float gf = ds_factor<T>(a, t.seq, kvh, HD);
        float lse = INFINITY, d = 0.f;
        if (row < t.len) {
            const long long at = (long long)head * a.tokens + t.start + row;
            lse = a.lse[at];
            lse = lse == -INFINITY ? INFINITY : lse * kLog2e;
            d = a.delta[at] * gf;
        }
        bool ok = true;
        for (int j = 0; j < n; ++j) {
            const uint32_t s0 = tS + lanes + 128 * (j & 1) + 64 * half;
            ok = bar_wait(s_ready + (j & 1), (j / 2) & 1, gone);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            const int lim = min(t.len, a.causal ? row + 1 : t.len) - j * kTile - 64 * half;   // columns below are seen
            float2 p[32];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t s[32];
                ld32(s, s0 + 32 * b);
                wait_ld();
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    p[16 * b + x] = exp2_both(__ffma2_rn(pair(s[2 * x], s[2 * x + 1]), both(a.c), both(-lse)));
            }
            ok = bar_wait(dp_ready, j & 1, gone);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            const bool part = __any_sync(0xffffffffu, lim < 64);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t s[32], w[16];
                ld32(s, p0 + 32 * b);
                wait_ld();
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    float2 e = __fmul2_rn(p[16 * b + x], __ffma2_rn(pair(s[2 * x], s[2 * x + 1]), both(gf), both(-d)));
                    if (part) {
                        if (32 * b + 2 * x >= lim) e.x = 0.f;
                        if (32 * b + 2 * x + 1 >= lim) e.y = 0.f;
                    }
                    w[x] = pack2<T>(e.x, e.y);
                }
                st16(s0 + 16 * b, w);
            }
            wait_st();
            fence_before();
            bar_arrive(ds_ready);
        }
        if (ok) ok = bar_wait(done, 0, gone);
        if (__all_sync(0xffffffffu, ok)) {
            fence_after();
            store_row<T, HD>(tQ + lanes, a.scale / gf, dq + row * out_row, row < t.len, half, 2);
        }
    }
    fence_before();
    __syncthreads();
    settle(gone);
    fence_after();
    if (warp == 8) tmem_free(tm, 512);
    if (threadIdx.x == 0 && *gone) atomicOr(a.err, kErrTcWait);
}

// One launch for both: the blocks of dq, shorter, fill the SMs that run out of dk
// and dv (two launches one after the other: 1022 against 1013 us for forward
// and backward of 8192 tokens).
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) k_packed_bwd_tc(const __grid_constant__ BwdArgs a, unsigned dkv_blocks) {
    extern __shared__ __align__(1024) uint8_t sm[];
    if (blockIdx.x < dkv_blocks) block_dkv<T, HD>(a, sm, blockIdx.x);
    else block_dq<T, HD>(a, sm, blockIdx.x - dkv_blocks, gridDim.x - dkv_blocks);
}

// D = do . o of the rows of a tile of one head, HD / 8 lanes a row; in a
// sequence's first tile o is the sum of what was stored and what rounding took
// from it.  float16: the largest |do| and |v| of its key/value head (blocks of y = 1 read v).  Every
// row of a thread is read before the first is summed.
template <typename T, int HD>
__global__ void __launch_bounds__(256) k_packed_delta16(const PackedParams p, float* __restrict__ delta,
                                                        float* __restrict__ top) {
    constexpr int L = HD / 8, STEP = 256 / L, N = kTile / STEP;
    const bool is_v = blockIdx.y;
    const int heads = is_v ? p.kv_heads : p.heads, head = blockIdx.x % p.heads, lane = threadIdx.x % L;
    if (head >= heads) return;
    const PackedTile t = packed_tile(p.cu, p.n_seqs, p.tokens, kTile, blockIdx.x / p.heads);
    if (t.row0 >= t.len || t.seq == p.n_seqs) return;
    const Rows& x = is_v ? p.v : p.dout;
    const T* in = static_cast<const T*>(x.p) + t.start * x.row + head * x.head + lane * 8;
    const long long at = (t.start * p.heads + head) * HD + lane * 8, row = (long long)p.heads * HD;
    const bool fine = p.low && t.row0 == 0;
    uint4 g[N], o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = t.row0 + threadIdx.x / L + i * STEP;
        g[i] = o[i] = make_uint4(0, 0, 0, 0);
        if (r < t.len) {
            g[i] = *reinterpret_cast<const uint4*>(in + r * x.row);
            if (!is_v) o[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.out_in) + at + r * row);
        }
    }
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = t.row0 + threadIdx.x / L + i * STEP;
        const T *ge = reinterpret_cast<const T*>(&g[i]), *oe = reinterpret_cast<const T*>(&o[i]);
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            m = fmaxf(m, fabsf(to_f32(ge[k])));
            s = fmaf(to_f32(ge[k]), to_f32(oe[k]), s);
        }
        if (fine && !is_v && r < t.len) {
            const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.low) + at + r * row);
            const T* ue = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int k = 0; k < 8; ++k) s = fmaf(to_f32(ge[k]), to_f32(ue[k]), s);
        }
#pragma unroll
        for (int off = L / 2; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        if (r < t.len && !is_v && lane == 0) delta[head * p.tokens + t.start + r] = s;
    }
    if (std::is_same<T, __half>::value) {
        const int kvh = is_v ? head : head / (p.heads / p.kv_heads);
        int* at = reinterpret_cast<int*>(top + 2 * ((long long)t.seq * p.kv_heads + kvh) + is_v);
#pragma unroll
        for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
        if ((threadIdx.x & 31) == 0 && m > 0.f) atomicMax(at, __float_as_int(m));      // a maximum: any order gives it
    }
}

template <typename T, int HD>
int launch_bwd(const BwdArgs& a, const PackedParams& p, cudaStream_t s) {
    using Sh = Shape<HD>;
    const bool f16 = std::is_same<T, __half>::value;
    float* top = const_cast<float*>(a.top);
    if (f16 && cudaMemsetAsync(top, 0, sizeof(float) * 2 * p.n_seqs * p.kv_heads, s) != cudaSuccess) return kErrCuda;
    const unsigned slots = (unsigned)packed_slots(a.tokens, a.n_seqs, kTile);
    k_packed_delta16<T, HD><<<dim3(slots * a.heads, f16 ? 2 : 1), 256, 0, s>>>(p, const_cast<float*>(a.delta), top);
    if (cudaGetLastError() != cudaSuccess) return kErrCuda;
    if (!allow_smem<&k_packed_bwd_tc<T, HD>>(Sh::SMEM)) return kErrCuda;
    k_packed_bwd_tc<T, HD><<<slots * (a.kv_heads + a.heads), kThreads, Sh::SMEM, s>>>(a, slots * a.kv_heads);
    return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

template <typename T>
int bwd_by_dim(const BwdArgs& a, const PackedParams& p, cudaStream_t s) {
    switch (p.head_dim) {
        case 32: return launch_bwd<T, 32>(a, p, s);
        case 64: return launch_bwd<T, 64>(a, p, s);
        default: return launch_bwd<T, 128>(a, p, s);
    }
}

}  // namespace

// Workspace: D [heads, tokens], then the largest values [n_seqs, kv_heads, 2].
int attention_packed_backward_tc(const PackedParams& p, cudaStream_t s) {
    BwdArgs a{};
    if (!rows_map(&a.q, p.q, p.type, p.tokens, p.heads, p.head_dim) ||
        !rows_map(&a.k, p.k, p.type, p.tokens, p.kv_heads, p.head_dim) ||
        !rows_map(&a.v, p.v, p.type, p.tokens, p.kv_heads, p.head_dim) ||
        !rows_map(&a.g, p.dout, p.type, p.tokens, p.heads, p.head_dim))
        return kErrUnsupported;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return kErrCuda; }
    a.cu = p.cu; a.n_seqs = p.n_seqs; a.heads = p.heads; a.kv_heads = p.kv_heads; a.group = p.heads / p.kv_heads;
    a.causal = p.causal; a.tokens = p.tokens;
    a.c = p.scale == 0.f ? 1e-30f : p.scale * kLog2e;
    a.scale = p.scale;
    a.lse = p.lse_in;
    a.delta = static_cast<float*>(p.ws);
    a.top = a.delta + p.tokens * p.heads;
    a.dq = p.dq; a.dk = p.dk; a.dv = p.dv;
    a.err = device_error_word(dev);
    if (!a.err) return kErrCuda;
    return p.type == kBF16 ? bwd_by_dim<__nv_bfloat16>(a, p, s) : bwd_by_dim<__half>(a, p, s);
}

}  // namespace racb
