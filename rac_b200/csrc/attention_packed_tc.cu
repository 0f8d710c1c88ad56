// attention_packed_tc.cu -- attention over packed prompts on the tensor cores,
// float16 and bfloat16, forward.
//
// A block has two tiles of 128 query rows of one head.  Per tile of 128 keys:
// S = Q K^T (shared memory times shared memory) into tensor memory; a thread a
// row takes the scores to registers, keeps a running maximum and sum, and puts
// the weights, rounded to the type, over the scores; O += P V takes them from
// there.  The two query tiles have a softmax warpgroup each, and while one
// weighs, the matrix unit works for the other.  Keys and values come by TMA
// into a ring.  The weights' rounding is half a step of the type, like the
// output's own, and in float16 at most 2^-25 of the largest weight where they
// are subnormal; sums and statistics are 32-bit.
//
// Bound: 512 cycles of the matrix unit for each of a tile's two products against
// some 1500 of softmax instructions, which the turn-taking hides; what is left
// is the way from weights to product to the next scores.  13 k tokens of 32 x
// 128 heads, causal: 0.76 ms, 1000 TFLOP/s, 0.60 of the measured bf16 peak.
#include "attn_common.cuh"
#include "tensor_core.cuh"

namespace racb {
namespace {

using namespace tc;

constexpr int kRows = 128;                 // query rows of a tile: one lane of tensor memory each
constexpr int kKeys = 128;                 // keys of a tile
// Warps 0-3, 4-7: softmax of query tile 0, 1; 8: matrix instructions; 9: loads; 10, 11 fill the warpgroup.
constexpr int kThreads = 384;
// Registers: 168 x 384 at launch = 216 x 256 + 72 x 128.
constexpr int kLaunchRegs = 168, kSoftmaxRegs = 216, kOtherRegs = 72;
static_assert(kSoftmaxRegs * 256 + kOtherRegs * 128 <= kLaunchRegs * kThreads, "register split");

struct FwdArgs {
    CUtensorMap q, k, v;
    const int* cu;
    int n_seqs, heads, group, causal, zero_rest;
    long long tokens;
    float c;                               // scale * log2(e)
    void *out, *low;
    float* lse;
    unsigned int* err;
};

template <int HD>
struct Shape {
    static constexpr int SW = HD * 2 < 128 ? HD * 2 : 128;          // swizzled row, bytes
    static constexpr int BOXES = HD * 2 / SW;
    static constexpr int BOX = kRows * SW;                          // bytes of a box of 128 rows
    static constexpr int TILE = BOXES * BOX;
    static constexpr int STAGES = HD == 128 ? 5 : 6;
    static constexpr int SMEM = 1024 + (2 + STAGES) * TILE;
    // tensor memory columns
    static constexpr int S0 = 0, O0 = 256;
};

// FINE: the first key tile's weights, which the first rows have no others beside,
// in two parts, and what rounding takes from those rows' output.  A kernel of its
// own: decided at run time it cost the calls without it 810 us for 650 (13 k tokens).
template <typename T, int HD, bool FINE>
__global__ void __launch_bounds__(kThreads, 1) k_packed_fwd_tc(const __grid_constant__ FwdArgs a) {
    using Sh = Shape<HD>;
    constexpr int ST = Sh::STAGES;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t q_full[2], full[ST], empty[ST], fixed, s_ready[2], p_ready[2], o_ready[2];
    __shared__ uint32_t tmem_base;
    __shared__ int gone;
    uint8_t* base = raw + ((1024 - (smem(raw) & 1023)) & 1023);
    uint8_t* qs = base;
    uint8_t* ring = base + 2 * Sh::TILE;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int head = blockIdx.x % a.heads, kvh = head / a.group;
    const PackedTile t = packed_tile(a.cu, a.n_seqs, a.tokens, 2 * kRows, (gridDim.x - 1 - blockIdx.x) / a.heads);
    if (t.row0 >= t.len) return;
    T* out = static_cast<T*>(a.out) + (t.start * a.heads + head) * HD;
    T* low = static_cast<T*>(a.low) + (t.start * a.heads + head) * HD;
    const long long out_row = (long long)a.heads * HD;
    if (t.seq == a.n_seqs) {                  // behind the last sequence
        if (a.zero_rest) {
            const int n = min(2 * kRows, t.len - t.row0) * (HD / 8);
            for (int e = threadIdx.x; e < n; e += kThreads)
                *reinterpret_cast<uint4*>(out + (t.row0 + e / (HD / 8)) * out_row + (e % (HD / 8)) * 8) =
                    make_uint4(0, 0, 0, 0);
        }
        return;
    }
    // Key tiles of the two query tiles; the second has none where it has no rows.
    int n_tiles[2];
    for (int w = 0; w < 2; ++w) {
        const int r = t.row0 + w * kRows;
        const int last = a.causal ? min(r + kRows, t.len) : t.len;
        n_tiles[w] = r < t.len ? (last + kKeys - 1) / kKeys : 0;
    }
    const int n = max(n_tiles[0], n_tiles[1]);
    const bool ragged = n * kKeys > t.len;    // the last key tile runs into the next sequence

    // The loading thread sets up the barriers and sends for the first tiles while
    // tensor memory is allocated: a block's first product waits for little else.
    if (threadIdx.x == 32 * 9) {
        gone = 0;
        bar_init(&q_full[0], 1);
        bar_init(&q_full[1], 1);
        bar_init(&fixed, 1);
        for (int i = 0; i < ST; ++i) { bar_init(&full[i], 1); bar_init(&empty[i], 1); }
        for (int w = 0; w < 2; ++w) { bar_init(&s_ready[w], 1); bar_init(&p_ready[w], kRows); bar_init(&o_ready[w], 1); }
        bar_init_done();
        for (int w = 0; w < 2 && n_tiles[w]; ++w) {
            bar_expect(&q_full[w], Sh::TILE);
            for (int b = 0; b < Sh::BOXES; ++b)
                load_3d(qs + w * Sh::TILE + b * Sh::BOX, &a.q, b * (Sh::SW / 2), head, (int)t.start + t.row0 + w * kRows,
                        &q_full[w]);
            if (w) break;
            bar_expect(&full[0], Sh::TILE);
            for (int b = 0; b < Sh::BOXES; ++b)
                load_3d(ring + b * Sh::BOX, &a.k, b * (Sh::SW / 2), kvh, (int)t.start, &full[0]);
        }
    }
    if (warp == 8) tmem_alloc(&tmem_base, 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm = tmem_base;

    if (warp >= 8) {
    fewer_registers<kOtherRegs>();
    if (warp == 9) {
        // ── loads: K0, V0, K1, V1, ... through the ring ──
        if (lane == 0) {
            for (int i = 1; i < 2 * n; ++i) {
                const int st = i % ST;
                if (i >= ST && !bar_wait(&empty[st], (i / ST - 1) & 1, &gone)) break;
                bar_expect(&full[st], Sh::TILE);
                for (int b = 0; b < Sh::BOXES; ++b)
                    load_3d(ring + st * Sh::TILE + b * Sh::BOX, i & 1 ? &a.v : &a.k, b * (Sh::SW / 2), kvh,
                            (int)t.start + (i >> 1) * kKeys, &full[st]);
            }
        }
        __syncwarp();
        if (ragged) {
            // Rows of the last V tile that are another sequence's: their weight
            // is 0, and 0 times their NaN would not be.
            const int i = 2 * n - 1, st = i % ST;
            if (bar_wait(&full[st], (i / ST) & 1, &gone)) {
                const int r0 = t.len - (n - 1) * kKeys;
                constexpr int U = Sh::SW / 16;
                for (int e = lane; e < (kKeys - r0) * U * Sh::BOXES; e += 32) {
                    const int b = e / ((kKeys - r0) * U), x = e % ((kKeys - r0) * U);
                    *reinterpret_cast<uint4*>(ring + st * Sh::TILE + b * Sh::BOX + r0 * Sh::SW + x * 16) =
                        make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();
            }
            __syncwarp();
            if (lane == 0) bar_arrive(&fixed);
        }
    } else if (warp == 8) {
        // ── matrix instructions, one thread ──
        if (lane == 0) {
            constexpr uint32_t iqk = instruction<T>(kRows, kKeys, false), ipv = instruction<T>(kRows, HD, true);
            auto scores = [&](int w, int i) {           // S_w = Q_w K^T, K in ring entry i
                product_ss<HD / 16, Sh::SW>(tm + Sh::S0 + w * kKeys, smem(qs + w * Sh::TILE), smem(ring + (i % ST) * Sh::TILE),
                                            Sh::BOX, iqk);
                commit(&s_ready[w]);
            };
            bool ok = bar_wait(&full[0], 0, &gone);
            for (int w = 0; ok && w < 2; ++w) {
                if (!n_tiles[w]) continue;
                ok = bar_wait(&q_full[w], 0, &gone);
                if (ok) scores(w, 0);
            }
            if (ok) commit(&empty[0]);
            for (int j = 0; ok && j < n; ++j) {
                const int vi = 2 * j + 1, ki = 2 * j + 2;
                ok = bar_wait(&full[vi % ST], (vi / ST) & 1, &gone);
                if (ok && ragged && j == n - 1) ok = bar_wait(&fixed, 0, &gone);
                if (ok && j + 1 < n) ok = bar_wait(&full[ki % ST], (ki / ST) & 1, &gone);
                for (int w = 0; ok && w < 2; ++w) {
                    if (j >= n_tiles[w]) continue;
                    ok = bar_wait(&p_ready[w], j & 1, &gone);
                    if (!ok) break;
                    fence_after();
                    const uint64_t vb = operand<Sh::SW>(smem(ring + (vi % ST) * Sh::TILE), Sh::BOX, 8 * Sh::SW);
                    const bool fine = FINE && j == 0;        // the weights' second parts, 64 columns on
                    if (fine) {
#pragma unroll
                        for (int k = 0; k < kKeys; k += 16)
                            mma_ts(tm + Sh::O0 + w * HD, tm + Sh::S0 + w * kKeys + 64 + k / 2, vb + (k * Sh::SW >> 4), ipv, k > 0);
                    }
#pragma unroll
                    for (int k = 0; k < kKeys; k += 16)
                        mma_ts(tm + Sh::O0 + w * HD, tm + Sh::S0 + w * kKeys + k / 2, vb + (k * Sh::SW >> 4), ipv,
                               j > 0 || k > 0 || fine);
                    if (j + 1 < n_tiles[w]) scores(w, ki);
                    else commit(&o_ready[w]);
                }
                if (!ok) break;
                commit(&empty[vi % ST]);
                if (j + 1 < n) commit(&empty[ki % ST]);
            }
        }
        __syncwarp();
    }
    } else {
    more_registers<kSoftmaxRegs>();
    if (n_tiles[warp >> 2]) {
        // ── softmax: a thread a row ──
        const int w = warp >> 2, row = t.row0 + w * kRows + (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tm + lanes + Sh::S0 + w * kKeys, to = tm + lanes + Sh::O0 + w * HD;
        const bool neg = a.c < 0.f;
        float m = 0.f, l = 0.f;               // weights are exp2(c s - m)
        bool ok = true;
        for (int j = 0; j < n_tiles[w]; ++j) {
            ok = bar_wait(&s_ready[w], j & 1, &gone);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            uint32_t s[4][32];
#pragma unroll
            for (int b = 0; b < 4; ++b) ld32(s[b], ts + 32 * b);
            wait_ld();
            const int lim = min(t.len, a.causal ? row + 1 : t.len) - j * kKeys;     // keys below are seen
            if (__any_sync(0xffffffffu, lim < kKeys)) {
                const uint32_t hide = neg ? 0x7f800000u : 0xff800000u;
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (32 * b + i >= lim) s[b][i] = hide;
            }
            float x[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) x[b] = neg ? smallest32(s[b]) : largest32(s[b]);
            float top = (neg ? fminf(fminf(x[0], x[1]), fminf(x[2], x[3])) : fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))) * a.c;
            if (top == -INFINITY) top = j ? m : 0.f;
            // The reference point moves only when a weight would pass 2^8: most
            // tiles leave the sums where they are.
            if (j == 0) {
                m = top;
            } else if (__any_sync(0xffffffffu, top > m + 8.f)) {
                const float up = top > m + 8.f ? exp2_fast(m - top) : 1.f;
                if (top > m + 8.f) m = top;
                l *= up;
#pragma unroll
                for (int b = 0; b < HD / 32; ++b) {
                    uint32_t o[32];
                    ld32(o, to + 32 * b);
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * up);
                    st32(to + 32 * b, o);
                }
            }
            const float2 c2 = both(a.c), m2 = both(-m);
            float2 add[2] = {both(0.f), both(0.f)};
            if (FINE && j == 0) {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t p[16], d[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 e = exp2_both(__ffma2_rn(pair(s[b][2 * i], s[b][2 * i + 1]), c2, m2));
                        add[i & 1] = __fadd2_rn(add[i & 1], e);
                        p[i] = pack2<T>(e.x, e.y);
                        d[i] = pack2<T>(e.x - low_of<T>(p[i]), e.y - high_of<T>(p[i]));
                    }
                    st16(ts + 16 * b, p);
                    st16(ts + 64 + 16 * b, d);
                }
            } else {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 e = exp2_both(__ffma2_rn(pair(s[b][2 * i], s[b][2 * i + 1]), c2, m2));
                        add[i & 1] = __fadd2_rn(add[i & 1], e);
                        p[i] = pack2<T>(e.x, e.y);
                    }
                    st16(ts + 16 * b, p);
                }
            }
            l += (add[0].x + add[0].y) + (add[1].x + add[1].y);
            wait_st();
            fence_before();
            bar_arrive(&p_ready[w]);
        }
        if (ok) ok = bar_wait(&o_ready[w], 0, &gone);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
            fence_after();
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int b = 0; b < HD / 32; ++b) {
                uint32_t o[32];
                ld32(o, to + 32 * b);
                wait_ld();
                if (row < t.len) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint4 u;
                        u.x = pack2<T>(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
                        u.y = pack2<T>(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
                        u.z = pack2<T>(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
                        u.w = pack2<T>(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
                        *reinterpret_cast<uint4*>(out + row * out_row + 32 * b + i) = u;
                        if (FINE && row < kRows) {
                            const uint32_t h[4] = {u.x, u.y, u.z, u.w};
                            uint32_t d[4];
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                d[y] = pack2<T>(__uint_as_float(o[i + 2 * y]) * inv - low_of<T>(h[y]),
                                                __uint_as_float(o[i + 2 * y + 1]) * inv - high_of<T>(h[y]));
                            *reinterpret_cast<uint4*>(low + row * out_row + 32 * b + i) = make_uint4(d[0], d[1], d[2], d[3]);
                        }
                    }
                }
            }
            if (a.lse && row < t.len)
                a.lse[(long long)head * a.tokens + t.start + row] =
                    l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
        }
    }
    }
    fence_before();
    __syncthreads();
    settle(&gone);
    fence_after();
    if (warp == 8) tmem_free(tm, 512);
    if (threadIdx.x == 0 && gone) atomicOr(a.err, kErrTcWait);
}

template <typename T, int HD>
int launch_fwd(const FwdArgs& a, cudaStream_t s) {
    const unsigned grid = (unsigned)(packed_slots(a.tokens, a.n_seqs, 2 * kRows) * a.heads);
    if (a.low) {
        if (!allow_smem<&k_packed_fwd_tc<T, HD, true>>(Shape<HD>::SMEM)) return kErrCuda;
        k_packed_fwd_tc<T, HD, true><<<grid, kThreads, Shape<HD>::SMEM, s>>>(a);
    } else {
        if (!allow_smem<&k_packed_fwd_tc<T, HD, false>>(Shape<HD>::SMEM)) return kErrCuda;
        k_packed_fwd_tc<T, HD, false><<<grid, kThreads, Shape<HD>::SMEM, s>>>(a);
    }
    return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

template <typename T>
int fwd_by_dim(const FwdArgs& a, int hd, cudaStream_t s) {
    switch (hd) {
        case 32: return launch_fwd<T, 32>(a, s);
        case 64: return launch_fwd<T, 64>(a, s);
        default: return launch_fwd<T, 128>(a, s);
    }
}

}  // namespace

// Rows of heads as a [tokens, heads, head_dim] tensor map with boxes of 128 rows of one head.
bool rows_map(CUtensorMap* m, const Rows& r, int type, long long tokens, int heads, int hd) {
    const int e = elem_bytes(type), sw = hd * e < 128 ? hd * e : 128;
    const uint64_t dims[3] = {(uint64_t)hd, (uint64_t)heads, (uint64_t)tokens};
    // An axis of one place is never stepped along.
    const uint64_t strides[2] = {(uint64_t)(heads > 1 ? r.head : hd) * e, (uint64_t)(tokens > 1 ? r.row : (long long)heads * hd) * e};
    const uint32_t box[3] = {(uint32_t)(sw / e), 1, (uint32_t)kRows};
    return encode_tensor(m, type == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, r.p,
                         dims, strides, box, sw);
}

int attention_packed_tc(const PackedParams& p, cudaStream_t s) {
    FwdArgs a{};
    if (!rows_map(&a.q, p.q, p.type, p.tokens, p.heads, p.head_dim) ||
        !rows_map(&a.k, p.k, p.type, p.tokens, p.kv_heads, p.head_dim) ||
        !rows_map(&a.v, p.v, p.type, p.tokens, p.kv_heads, p.head_dim))
        return kErrUnsupported;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return kErrCuda; }
    a.cu = p.cu; a.n_seqs = p.n_seqs; a.heads = p.heads; a.group = p.heads / p.kv_heads; a.causal = p.causal;
    a.zero_rest = p.zero_rest; a.tokens = p.tokens; a.out = p.out; a.lse = p.lse; a.low = p.low;
    // 0 would turn a hidden score's infinity into NaN; 1e-30 weighs the rest alike.
    a.c = p.scale == 0.f ? 1e-30f : p.scale * 1.4426950408889634f;
    a.err = device_error_word(dev);
    if (!a.err) return kErrCuda;
    return p.type == kBF16 ? fwd_by_dim<__nv_bfloat16>(a, p.head_dim, s) : fwd_by_dim<__half>(a, p.head_dim, s);
}

}  // namespace racb
