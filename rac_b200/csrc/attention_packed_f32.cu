// attention_packed_f32.cu -- attention over packed prompts in float32, forward
// and backward, on the float16 tensor cores.
//
// A float32 value x is kept as two float16 parts, hi = f16(x f) and lo =
// f16(x f - hi), 22 bits together; f is a power of two for each head of each
// tile of 128 rows that puts the tile's largest value between 2^13 and 2^14,
// so that the error is 2^-22 of a value or 2^-39 of its tile's largest.  A
// product of two such matrices is lo hi + hi lo + hi hi (lo lo lies below the
// last bit): three float16 products, a rate of 1647 / 3 = 549 TFLOP/s against
// the FP32 pipe's 74.
//
// The tensor core adds into its 32-bit sums by cutting off (measured: 1e-7 of
// the sum for each instruction of 16 summed values, all in one direction, so
// that 1024 of them lose 1e-4).  So a sum in tensor memory is never carried on
// from one tile to the next: it is added to 32-bit registers, rounded to
// nearest, where the tile's factor is applied as well.  Within a product the
// small parts come first.
//
// Bound: the three products of each pair of tiles, and between them the way of
// every partial sum through registers.  4096 tokens in ragged causal prompts, 32
// heads of 128 with keys of their own: 288 us, of them 68 for the parts (87 us is
// what the products alone need); 2048 tokens, 16 heads of 64 on 4, both ways, forward and backward:
// 180 us; one by one splitting takes 9 and 17, the forward 44, dq, dk and dv 118, the
// heads' sums 7.
#include "attn_common.cuh"
#include "tensor_core.cuh"

namespace racb {
namespace {

using namespace tc;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSplit = 128;                // rows that share a factor
constexpr int kWide = 128, kBoxRows = 64;  // rows of a tile that stays in place, of a TMA box
// A product of 64 columns takes the matrix unit as long as one of 128 (64 cycles
// an instruction), so that the tiles that pass by have 128 rows as well, except
// in the backward kernels at dim 128, which have no room for them.
template <int HD> constexpr int narrow() { return HD == 128 ? 64 : 128; }

// ── parts ─────────────────────────────────────────────────────────────────
struct SplitArgs {
    Rows in[4];                            // q, k, v, dout
    int heads[4], first[5];                // heads of each; prefix sums
    __half* parts[4];                      // [tokens, 2 heads, dim]: hi of each head, then lo
    float* factors[4];                     // [slots, heads]: 1 / f
    float *vnorm, *gnorm;                  // with dout: like v's and dout's factors, the largest |v f| and |do f| of a row
    const float* out;                      // with dout: the forward's output, for D = do . o
    float *delta, *dtop;                   // [heads, tokens]; like dout's factors, the largest |D|
    const int* cu;
    int n_seqs;
    int negate;                            // q's parts are those of -q (a negative scale: the kernels take its size)
    long long tokens;
};

template <int HD>
__global__ void __launch_bounds__(256) k_split(const SplitArgs a) {
    constexpr int L = HD / 4, STEP = 256 / L, N = kSplit / STEP;
    __shared__ float red[8], red2[2][8];
    int h = blockIdx.x % a.first[4], w = 0;
    const int slot = blockIdx.x / a.first[4];
    while (h >= a.first[w + 1]) ++w;
    h -= a.first[w];
    const PackedTile t = packed_tile(a.cu, a.n_seqs, a.tokens, kSplit, slot);
    if (t.row0 >= t.len || t.seq == a.n_seqs) return;
    const int lane = threadIdx.x % L, row0 = t.row0 + threadIdx.x / L;
    const float* in = static_cast<const float*>(a.in[w].p) + t.start * a.in[w].row + h * a.in[w].head + lane * 4;
    float4 x[N];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = row0 + i * STEP;
        x[i] = r < t.len ? *reinterpret_cast<const float4*>(in + r * a.in[w].row) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float y[4] = {fabsf(x[i].x), fabsf(x[i].y), fabsf(x[i].z), fabsf(x[i].w)};
#pragma unroll
        for (int k = 0; k < 4; ++k) m = y[k] < INFINITY ? fmaxf(m, y[k]) : m;    // infinities and NaN keep to themselves
    }
    float dtop = 0.f;
    if (w == 3) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row0 + i * STEP;
            float s = 0.f;
            if (r < t.len) {
                const float4 o = *reinterpret_cast<const float4*>(a.out + ((t.start + r) * a.heads[3] + h) * HD + lane * 4);
                s = fmaf(x[i].x, o.x, fmaf(x[i].y, o.y, fmaf(x[i].z, o.z, x[i].w * o.w)));
            }
#pragma unroll
            for (int off = L / 2; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
            if (lane == 0 && r < t.len) a.delta[h * a.tokens + t.start + r] = s;
            if (fabsf(s) < INFINITY) dtop = fmaxf(dtop, fabsf(s));
        }
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, red[i]);
    int e = 14;
    if (m > 0.f) frexpf(m, &e);            // m < 2^e
    e = max(14 - e, -112);
    e = min(e, 120);
    const float f = ldexpf(w == 0 && a.negate ? -1.f : 1.f, e);
    if (threadIdx.x == 0) a.factors[w][(long long)slot * a.heads[w] + h] = ldexpf(1.f, -e);
    __half* p = a.parts[w] + (t.start * 2 * a.heads[w] + h) * HD + lane * 4;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int r = row0 + i * STEP;
        if (r >= t.len) continue;
        const float y[4] = {x[i].x * f, x[i].y * f, x[i].z * f, x[i].w * f};
        __half hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            hi[k] = __float2half_rn(y[k]);
            lo[k] = __float2half_rn(y[k] - __half2float(hi[k]));
        }
        __half* row = p + (long long)r * 2 * a.heads[w] * HD;
        *reinterpret_cast<uint2*>(row) = *reinterpret_cast<uint2*>(hi);
        *reinterpret_cast<uint2*>(row + (long long)a.heads[w] * HD) = *reinterpret_cast<uint2*>(lo);
    }
    if (w < 2 || !a.delta) return;
    // What bounds do . v and D, for the factors of dS.
    float norm = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float y[4] = {x[i].x * f, x[i].y * f, x[i].z * f, x[i].w * f};
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) s = fabsf(y[k]) < INFINITY ? fmaf(y[k], y[k], s) : s;
#pragma unroll
        for (int off = L / 2; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        norm = fmaxf(norm, s);
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) {
        norm = fmaxf(norm, __shfl_xor_sync(0xffffffffu, norm, off));
        dtop = fmaxf(dtop, __shfl_xor_sync(0xffffffffu, dtop, off));
    }
    if ((threadIdx.x & 31) == 0) {
        red2[0][threadIdx.x >> 5] = norm;
        red2[1][threadIdx.x >> 5] = dtop;
    }
    __syncthreads();
    if (threadIdx.x) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        norm = fmaxf(norm, red2[0][i]);
        dtop = fmaxf(dtop, red2[1][i]);
    }
    const long long at = (long long)slot * a.heads[w] + h;
    (w == 2 ? a.vnorm : a.gnorm)[at] = sqrtf(norm);
    if (w == 3) a.dtop[at] = dtop;
}

// ── tiles and products ────────────────────────────────────────────────────
struct Args {
    CUtensorMap q, k, v, g;                // boxes of 64 rows of one part of one head
    const int* cu;
    int n_seqs, heads, kv_heads, group, causal, zero_rest;
    long long tokens;
    float c, scale;                        // |scale| log2(e), scale
    int split;                             // dk, dv: one query head a block, to be added up
    const float *fq, *fk, *fv, *fg;        // factors
    const float *vnorm, *gnorm, *dtop;     // what bounds dS, see SplitArgs
    const __half *pq, *pk, *pv, *pg;       // parts
    const float *lse_in, *delta;
    float *out, *lse, *dq, *dk, *dv;
    unsigned int* err;
};

template <int HD>
struct Shape {
    static constexpr int SW = HD * 2 < 128 ? HD * 2 : 128;
    static constexpr int BOXES = HD * 2 / SW;
    // A part of a tile: its boxes of all rows; the other part behind it.
    static constexpr int part(int rows) { return rows * HD * 2; }
    static constexpr int tile(int rows) { return 2 * rows * HD * 2; }
};

// Both parts of a tile of ROWS rows (64 or 128): boxes [rows, SW] one after another.
template <int HD, int ROWS>
__device__ __forceinline__ void load_parts(uint8_t* dst, const CUtensorMap* m, int head, int heads, int row, uint64_t* bar) {
    using Sh = Shape<HD>;
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int b = 0; b < Sh::BOXES; ++b)
#pragma unroll
            for (int r = 0; r < ROWS; r += kBoxRows)
                load_3d(dst + part * ROWS * HD * 2 + (b * ROWS + r) * Sh::SW, m, b * (Sh::SW / 2), part * heads + head,
                        row + r, bar);
}

// Rows [r0, ROWS) of both parts become zeros, by one warp.
template <int HD, int ROWS>
__device__ __forceinline__ void zero_parts(uint8_t* tile, int r0) {
    using Sh = Shape<HD>;
    const int n = (ROWS - r0) * (Sh::SW / 16), lane = threadIdx.x & 31;
    for (int e = lane; e < n * Sh::BOXES * 2; e += 32)
        *reinterpret_cast<uint4*>(tile + (e / n) * ROWS * Sh::SW + r0 * Sh::SW + (e % n) * 16) = make_uint4(0, 0, 0, 0);
}

// D = A B^T over HD: A 128 rows, B N rows, both in parts.
template <int HD, int N>
__device__ __forceinline__ void parts_rows(uint32_t d, uint32_t a, uint32_t b) {
    using Sh = Shape<HD>;
    constexpr uint32_t instr = instruction<__half>(kWide, N, false);
#pragma unroll
    for (int t = 0; t < 3; ++t) {          // lo hi, hi lo, hi hi
        const uint64_t da = operand<Sh::SW>(a + (t == 0 ? Sh::part(kWide) : 0), 16, 8 * Sh::SW);
        const uint64_t db = operand<Sh::SW>(b + (t == 1 ? Sh::part(N) : 0), 16, 8 * Sh::SW);
#pragma unroll
        for (int k = 0; k < HD; k += 16)
            mma_ss(d, da + (((k * 2 / Sh::SW) * kWide * Sh::SW + (k * 2) % Sh::SW) >> 4),
                   db + (((k * 2 / Sh::SW) * N * Sh::SW + (k * 2) % Sh::SW) >> 4), instr, t > 0 || k > 0);
    }
}
// The same with A's rows in tensor memory: HD / 2 columns of hi, then of lo.
template <int HD, int N>
__device__ __forceinline__ void parts_rows_t(uint32_t d, uint32_t a, uint32_t b) {
    using Sh = Shape<HD>;
    constexpr uint32_t instr = instruction<__half>(kWide, N, false);
#pragma unroll
    for (int t = 0; t < 3; ++t) {
        const uint64_t db = operand<Sh::SW>(b + (t == 1 ? Sh::part(N) : 0), 16, 8 * Sh::SW);
#pragma unroll
        for (int k = 0; k < HD; k += 16)
            mma_ts(d, a + (t == 0 ? HD / 2 : 0) + k / 2, db + (((k * 2 / Sh::SW) * N * Sh::SW + (k * 2) % Sh::SW) >> 4),
                   instr, t > 0 || k > 0);
    }
}
// One part of a row, from global memory to the HD / 2 columns at addr of the thread's lane.
template <int HD>
__device__ __forceinline__ void put_row(uint32_t addr, const __half* row, bool live) {
#pragma unroll
    for (int b = 0; b < HD / 32; ++b) {
        uint32_t x[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 u = live ? *reinterpret_cast<const uint4*>(row + 32 * b + 8 * i) : make_uint4(0, 0, 0, 0);
            x[4 * i] = u.x; x[4 * i + 1] = u.y; x[4 * i + 2] = u.z; x[4 * i + 3] = u.w;
        }
        st16(addr + 16 * b, x);
    }
}
// D = W B: W [128, N] in tensor memory, for each 32 columns 16 of hi and 16 of
// lo; B N rows in parts, summed over.
template <int HD, int N>
__device__ __forceinline__ void parts_weights(uint32_t d, uint32_t w, uint32_t b) {
    using Sh = Shape<HD>;
    constexpr uint32_t instr = instruction<__half>(kWide, HD, true);
#pragma unroll
    for (int t = 0; t < 3; ++t) {
        const uint64_t db = operand<Sh::SW>(b + (t == 1 ? Sh::part(N) : 0), N * Sh::SW, 8 * Sh::SW);
#pragma unroll
        for (int k = 0; k < N; k += 16)
            mma_ts(d, w + (k / 32) * 32 + (k % 32) / 2 + (t == 0 ? 16 : 0), db + (k * Sh::SW >> 4), instr, t > 0 || k > 0);
    }
}
// 32 weights of a row as parts, to the columns that parts_weights reads.
__device__ __forceinline__ void put_parts(uint32_t addr, const float2* p) {
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        hi[i] = pack2<__half>(p[i].x, p[i].y);
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
        const float2 d = __ffma2_rn(h, both(-1.f), p[i]);
        lo[i] = pack2<__half>(d.x, d.y);
    }
    st16(addr, hi);
    st16(addr + 16, lo);
}
// acc += f * 32 columns.
__device__ __forceinline__ void take32(float2* acc, uint32_t addr, float f) {
    uint32_t o[32];
    ld32(o, addr);
    wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = __ffma2_rn(pair(o[2 * i], o[2 * i + 1]), both(f), acc[i]);
}
__device__ __forceinline__ void store32(float* dst, const float2* v, float f) {
#pragma unroll
    for (int i = 0; i < 16; i += 2)
        *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(v[i].x * f, v[i].y * f, v[i + 1].x * f, v[i + 1].y * f);
}
__device__ __forceinline__ void zero_rows_out(float* dst, long long row_stride, int hd, int row0, int len) {
    const int n = min(kWide, len - row0) * (hd / 4);
    for (int e = threadIdx.x; e < n; e += blockDim.x)
        *reinterpret_cast<float4*>(dst + (row0 + e / (hd / 4)) * row_stride + (e % (hd / 4)) * 4) =
            make_float4(0.f, 0.f, 0.f, 0.f);
}

// Warps 0-3, 4-7: mathematics; 8: matrix instructions; 9: loads; 10: row statistics.
constexpr int kThreads = 384;
constexpr int kLaunchRegs = 168, kMathRegs = 200, kOtherRegs = 104;
static_assert(kMathRegs * 256 + kOtherRegs * 128 <= kLaunchRegs * kThreads, "register split");

// Slot (of 128 rows) of a row of a sequence.
__device__ __forceinline__ long long slot_of(const PackedTile& t, int row) { return t.start / kSplit + t.seq + row / kSplit; }

// |scale| log2(e) times both tiles' factors: what a score of their parts is multiplied by.
// Neither 0, which would turn a hidden score's infinity into NaN, nor infinite, which would
// do so to a score of 0: a score of parts is below 2^36, and 1e-37 leaves it without weight.
__device__ __forceinline__ float score_factor(float cq, float fk) { return fminf(fmaxf(cq * fk, 1e-37f), 3e38f); }

constexpr int kKeysF32 = 128;              // keys of a tile, forward

// ── forward ───────────────────────────────────────────────────────────────
// The warpgroups take the key tiles in turn, each with its own scores, its own
// reference point and its own sum in registers; the two join at the end.
template <int HD>
struct FwdShape {
    using Sh = Shape<HD>;
    static constexpr int STAGES = HD == 128 ? 3 : 6, TILE = Sh::tile(kWide);
    static constexpr int BARS = STAGES * TILE, SMEM = BARS + 512;
    static_assert(STAGES * TILE >= kWide * (HD + 1) * 4 + kWide * 8, "room to join");
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) k_f32_fwd(const __grid_constant__ Args a) {
    using Sh = Shape<HD>;
    using Fs = FwdShape<HD>;
    constexpr int ST = Fs::STAGES, TILE = Fs::TILE;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint8_t* ring = sm;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Fs::BARS);
    uint64_t *full = bars, *empty = full + ST, *q_full = empty + ST, *fixed = q_full + 1, *s_ready = fixed + 1,
             *p_ready = s_ready + 2, *o_ready = p_ready + 2, *o_taken = o_ready + 2, *joined = o_taken + 1;
    uint32_t* tmem_base = reinterpret_cast<uint32_t*>(joined + 1);
    volatile int* gone = reinterpret_cast<volatile int*>(tmem_base + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int head = blockIdx.x % a.heads, kvh = head / a.group;
    const PackedTile t = packed_tile(a.cu, a.n_seqs, a.tokens, kWide, (gridDim.x - 1 - blockIdx.x) / a.heads);
    if (t.row0 >= t.len) return;
    float* out = a.out + (t.start * a.heads + head) * HD;
    const long long out_row = (long long)a.heads * HD;
    if (t.seq == a.n_seqs) {
        if (a.zero_rest) zero_rows_out(out, out_row, HD, t.row0, t.len);
        return;
    }
    const int last = a.causal ? min(t.row0 + kWide, t.len) : t.len;
    const int n = (last + kKeysF32 - 1) / kKeysF32;
    const bool ragged = n * kKeysF32 > t.len;

    if (threadIdx.x == 0) {
        *gone = 0;
        for (int i = 0; i < ST; ++i) { bar_init(full + i, 1); bar_init(empty + i, 1); }
        bar_init(q_full, 256); bar_init(fixed, 1); bar_init(joined, 128); bar_init(o_taken, 128);
        for (int w = 0; w < 2; ++w) { bar_init(s_ready + w, 1); bar_init(p_ready + w, 128); bar_init(o_ready + w, 1); }
        bar_init_done();
    }
    if (warp == 8) tmem_alloc(tmem_base, 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm = *tmem_base, tS = tm, tO = tm + 256, tQ = tm + 384;     // S twice; O; Q: both parts

    // The ring holds K0, K1, V0, K2, V1, K3, ...: entry of K_j, of V_j.
    auto k_entry = [](int j) { return j < 2 ? j : 2 * j - 1; };
    auto v_entry = [&](int j) { return n == 1 ? 1 : j + 2 < n + 1 ? 2 * j + 2 : n + j; };

    if (warp >= 8) {
        fewer_registers<kOtherRegs>();
        if (warp == 9) {
            if (lane == 0) {
                const int r0 = (int)t.start;
                int e = 0;
                bool ok = true;
                auto load = [&](const CUtensorMap* m, int j) {
                    const int st = e % ST;
                    if (e >= ST) ok = bar_wait(empty + st, (e / ST - 1) & 1, gone);
                    if (!ok) return;
                    bar_expect(full + st, TILE);
                    load_parts<HD, kKeysF32>(ring + st * TILE, m, kvh, a.kv_heads, r0 + j * kKeysF32, full + st);
                    ++e;
                };
                load(&a.k, 0);
                if (ok && n > 1) load(&a.k, 1);
                for (int j = 0; ok && j < n; ++j) {
                    load(&a.v, j);
                    if (ok && j + 2 < n) load(&a.k, j + 2);
                }
            }
            __syncwarp();
            if (ragged) {
                const int e = v_entry(n - 1), st = e % ST;
                if (bar_wait(full + st, (e / ST) & 1, gone)) {
                    zero_parts<HD, kKeysF32>(ring + st * TILE, t.len - (n - 1) * kKeysF32);
                    fence_async_smem();
                }
                __syncwarp();
                if (lane == 0) bar_arrive(fixed);
            }
        } else if (warp == 8) {
            if (lane == 0) {
                auto scores = [&](int j) {
                    const int e = k_entry(j), st = e % ST;
                    if (!bar_wait(full + st, (e / ST) & 1, gone)) return false;
                    parts_rows_t<HD, kKeysF32>(tS + 128 * (j & 1), tQ, smem(ring + st * TILE));
                    commit(s_ready + (j & 1));
                    commit(empty + st);
                    return true;
                };
                bool ok = bar_wait(q_full, 0, gone);
                fence_after();
                ok = ok && scores(0);
                if (ok && n > 1) ok = scores(1);
                for (int j = 0; ok && j < n; ++j) {
                    const int e = v_entry(j), st = e % ST, w = j & 1;
                    ok = bar_wait(full + st, (e / ST) & 1, gone) && (!(ragged && j == n - 1) || bar_wait(fixed, 0, gone)) &&
                         bar_wait(p_ready + w, (j >> 1) & 1, gone);
                    if (!ok) break;
                    // One block of sums: the other warpgroup has to have taken the last.
                    if (j) ok = bar_wait(o_taken, (j - 1) & 1, gone);
                    if (!ok) break;
                    fence_after();
                    parts_weights<HD, kKeysF32>(tO, tS + 128 * w, smem(ring + st * TILE));
                    commit(o_ready + w);
                    commit(empty + st);
                    if (j + 2 < n) ok = scores(j + 2);
                }
            }
            __syncwarp();
        }
    } else {
        more_registers<kMathRegs>();
        const int w = warp >> 2, lr = (warp & 3) * 32 + lane, row = t.row0 + lr;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, ts = tS + lanes + 128 * w, to = tO + lanes;
        put_row<HD>(tQ + lanes + w * (HD / 2), a.pq + ((t.start + row) * 2 * a.heads + w * a.heads + head) * HD, row < t.len);
        wait_st();
        fence_before();
        bar_arrive(q_full);
        const float cq = a.c * a.fq[slot_of(t, t.row0) * a.heads + head];
        float m = -INFINITY, l = 0.f;
        float2 o[HD / 2];
#pragma unroll
        for (int i = 0; i < HD / 2; ++i) o[i] = both(0.f);
        bool ok = true;
        for (int j = w; j < n; j += 2) {
            const long long ks = slot_of(t, j * kKeysF32) * a.kv_heads + kvh;
            const float c = score_factor(cq, a.fk[ks]), fv = a.fv[ks];
            ok = __all_sync(0xffffffffu, bar_wait(s_ready + w, (j >> 1) & 1, gone));
            if (!ok) break;
            fence_after();
            const int lim = min(t.len, a.causal ? row + 1 : t.len) - j * kKeysF32;     // keys below are seen
            const bool part = __any_sync(0xffffffffu, lim < kKeysF32);
            auto scores = [&](uint32_t (&x)[32], int b) {
                ld32(x, ts + 32 * b);
                wait_ld();
                if (part) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (32 * b + i >= lim) x[i] = 0xff800000u;
                }
            };
            // The scores are read twice, and the loops stay loops: what the warps run through
            // for a tile has to stay in the instruction cache.
            float y = -INFINITY;
#pragma unroll 1
            for (int b = 0; b < kKeysF32 / 32; ++b) {
                uint32_t x[32];
                scores(x, b);
                y = fmaxf(y, largest32(x));
            }
            const float top = y * c;
            // The reference point moves only when a weight would pass 2^8.
            if (top > m + 8.f) {
                const float up = exp2_fast(m - top);
                m = top;
                l *= up;
#pragma unroll
                for (int i = 0; i < HD / 2; ++i) o[i] = __fmul2_rn(o[i], both(up));
            }
            // Weights carry 2^6, which keeps their second parts above the smallest half.
            const float ref = m == -INFINITY ? 0.f : m - 6.f;
#pragma unroll 1
            for (int b = 0; b < kKeysF32 / 32; ++b) {
                uint32_t x[32];
                float2 p[16], add[2] = {both(0.f), both(0.f)};
                scores(x, b);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    p[i] = exp2_both(__ffma2_rn(pair(x[2 * i], x[2 * i + 1]), both(c), both(-ref)));
                    add[i & 1] = __fadd2_rn(add[i & 1], p[i]);
                }
                l += (add[0].x + add[0].y) + (add[1].x + add[1].y);
                put_parts(ts + 32 * b, p);
            }
            wait_st();
            fence_before();
            bar_arrive(p_ready + w);
            ok = __all_sync(0xffffffffu, bar_wait(o_ready + w, (j >> 1) & 1, gone));
            if (!ok) break;
            fence_after();
#pragma unroll
            for (int b = 0; b < HD / 32; ++b) take32(o + 16 * b, to + 32 * b, fv);
            fence_before();
            bar_arrive(o_taken);
        }
        // All products are done when both warpgroups are through: the ring is free.
        float* jo = reinterpret_cast<float*>(ring);
        float2* jm = reinterpret_cast<float2*>(jo + kWide * (HD + 1));
        if (w == 1) {
            if (ok && n > 1) {
                // The last product of the other warpgroup may still read the ring.
                ok = __all_sync(0xffffffffu, bar_wait(o_ready, ((n - 1) >> 1) & 1, gone));
                if (ok) {
                    jm[lr] = make_float2(m, l);
#pragma unroll
                    for (int i = 0; i < HD / 2; ++i) {
                        jo[lr * (HD + 1) + 2 * i] = o[i].x;
                        jo[lr * (HD + 1) + 2 * i + 1] = o[i].y;
                    }
                }
                bar_arrive(joined);
            }
        } else if (ok) {
            if (n > 1) {
                ok = __all_sync(0xffffffffu, bar_wait(joined, 0, gone));
                const float2 z = jm[lr];
                const float M = fmaxf(m, z.x), f0 = m == -INFINITY ? 0.f : exp2_fast(m - M),
                            f1 = z.x == -INFINITY ? 0.f : exp2_fast(z.x - M);
                l = l * f0 + z.y * f1;
                m = M;
#pragma unroll
                for (int i = 0; i < HD / 2; ++i)
                    o[i] = make_float2(o[i].x * f0 + jo[lr * (HD + 1) + 2 * i] * f1, o[i].y * f0 + jo[lr * (HD + 1) + 2 * i + 1] * f1);
            }
            if (ok && row < t.len) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
                for (int b = 0; b < HD / 32; ++b) store32(out + row * out_row + 32 * b, o + 16 * b, inv);
                if (a.lse)
                    a.lse[(long long)head * a.tokens + t.start + row] =
                        l == 0.f ? -INFINITY : (m - 6.f) * 0.69314718055994531f + logf(l);
            }
        }
    }
    fence_before();
    __syncthreads();
    settle(gone);
    fence_after();
    if (warp == 8) tmem_free(tm, 512);
    if (threadIdx.x == 0 && *gone) atomicOr(a.err, kErrTcWait);
}

// ── backward ──────────────────────────────────────────────────────────────
// For a tile of queries and one of keys  |dS| = P |do . v - D| <= B = max |do| max |v| +
// max |D|: rows of these two tiles bound do . v, and D, which holds the values of all the
// keys that a query sees, is bounded by itself.  dS goes into parts times a power of two g
// <= 2^15 / B (finite also where B is 0 or infinite) and P times 2^12:
// dS' = P' (acc f f' g 2^-12 - D g 2^-12), acc the sum of the parts of dO V^T and f, f'
// their factors.  B lies some 2^4 above a dO . V of independent values, so that dS of weights
// around 1 / n keeps 22 bits up to some 2^14 keys; a smaller one keeps 2^-40 of B.
constexpr float kPUp = 12.f, kPDown = 1.f / 4096.f;
struct DsFactors { float up, acc, down; };  // g; f f' g 2^-12; 1 / g
__device__ __forceinline__ DsFactors ds_factors(float fg, float gnorm, float dtop, float fv, float vnorm) {
    // The products' factors are powers of two: no rounding, and no overflow unless dS itself overflows.
    const float b = (gnorm * fg) * (vnorm * fv) + dtop;
    const int e = min(max((int)(__float_as_uint(b) >> 23) - 126, -111), 128);       // B < 2^e
    const float up = __uint_as_float((uint32_t)(142 - e) << 23);                     // 2^(15 - e)
    return {up, fminf(fg * up * fv, 3e38f) * kPDown, __uint_as_float((uint32_t)(112 + e) << 23)};
}

template <int HD>
struct BwdShape {
    using Sh = Shape<HD>;
    // Places of Q (dk/dv) or K (dq), which a later product reads again, and of dO or V.
    static constexpr int A = HD == 32 ? 3 : 2, B = HD == 128 ? 1 : 2;
    static constexpr int N = narrow<HD>(), TILE = Sh::tile(N), KEPT = Sh::tile(kWide);
    static constexpr int RING = 2 * KEPT, STAT = RING + (A + B) * TILE, BARS = STAT + 2 * 2 * N * 4 + 2 * 8;
    static constexpr int SMEM = BARS + 512;
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

// dk and dv of 128 keys: query tiles pass by, of all heads of the group.
// The order is dV(i), S(i+1), dK(i), dP(i+1); P(i) lies in S(i)'s columns, dS(i) in dP(i)'s.
template <int HD>
__device__ __forceinline__ void block_dkv(const Args& a, uint8_t* sm, unsigned block) {
    using Sh = Shape<HD>;
    using Bs = BwdShape<HD>;
    constexpr int NA = Bs::A, NB = Bs::B, N = Bs::N, TILE = Bs::TILE, C = N / 2;
    uint8_t *ks = sm, *vs = sm + Bs::KEPT, *qr = sm + Bs::RING, *gr = qr + NA * TILE;
    float* st_lse = reinterpret_cast<float*>(sm + Bs::STAT);       // negative; [2][64]
    float* st_d = st_lse + 2 * N;
    float2* st_ds = reinterpret_cast<float2*>(st_d + 2 * N);       // factors of dS: of acc, and back; [2]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Bs::BARS);
    uint64_t *q_full = bars, *q_empty = q_full + NA, *q_fixed = q_empty + NA, *g_full = q_fixed + NA, *g_empty = g_full + NB,
             *g_fixed = g_empty + NB, *kv_full = g_fixed + NB, *stat_full = kv_full + 2,
             *stat_empty = stat_full + 2, *s_ready = stat_empty + 2, *dp_ready = s_ready + 1, *p_ready = dp_ready + 1,
             *ds_ready = p_ready + 1, *dv_done = ds_ready + 1, *dk_done = dv_done + 1;
    uint32_t* tmem_base = reinterpret_cast<uint32_t*>(dk_done + 1);
    volatile int* gone = reinterpret_cast<volatile int*>(tmem_base + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // Sums of a group's heads, or of one of them.
    const int outs = a.split ? a.heads : a.kv_heads, each = a.split ? 1 : a.group;
    const int oh = block % outs, kvh = a.split ? oh / a.group : oh, head0 = oh * each;
    const PackedTile t = packed_tile(a.cu, a.n_seqs, a.tokens, kWide, block / outs);
    if (t.row0 >= t.len) return;
    const long long out_row = (long long)outs * HD;
    float* dk = a.dk + (t.start * outs + oh) * HD;
    float* dv = a.dv + (t.start * outs + oh) * HD;
    if (t.seq == a.n_seqs) {
        zero_rows_out(dk, out_row, HD, t.row0, t.len);
        zero_rows_out(dv, out_row, HD, t.row0, t.len);
        return;
    }
    const int first = a.causal ? t.row0 / N : 0;             // query tiles that see these keys
    const int nq = (t.len + N - 1) / N - first;
    const int n = nq * each;
    const bool ragged = t.len % N != 0;                      // the last query tile of each head

    // As in the 16-bit kernels, the first tiles are under way before the block meets.
    if (threadIdx.x == 32 * 9) {
        *gone = 0;
        for (int i = 0; i < NA; ++i) { bar_init(q_full + i, 1); bar_init(q_empty + i, 1); bar_init(q_fixed + i, 1); }
        for (int i = 0; i < NB; ++i) { bar_init(g_full + i, 1); bar_init(g_empty + i, 1); bar_init(g_fixed + i, 1); }
        bar_init(kv_full, 1);
        bar_init(kv_full + 1, 1);
        for (int i = 0; i < 2; ++i) { bar_init(stat_full + i, 1); bar_init(stat_empty + i, 256); }
        bar_init(s_ready, 1); bar_init(dp_ready, 1); bar_init(p_ready, 256); bar_init(ds_ready, 256);
        bar_init(dv_done, 1); bar_init(dk_done, 1);
        bar_init_done();
        const int k0 = (int)t.start + t.row0, q0 = (int)t.start + first * N;
        bar_expect(kv_full, Bs::KEPT);
        load_parts<HD, kWide>(ks, &a.k, kvh, a.kv_heads, k0, kv_full);
        bar_expect(q_full, TILE);
        load_parts<HD, N>(qr, &a.q, head0, a.heads, q0, q_full);
        bar_expect(kv_full + 1, Bs::KEPT);
        load_parts<HD, kWide>(vs, &a.v, kvh, a.kv_heads, k0, kv_full + 1);
        bar_expect(g_full, TILE);
        load_parts<HD, N>(gr, &a.g, head0, a.heads, q0, g_full);
    }
    if (warp == 8) tmem_alloc(tmem_base, 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm = *tmem_base, tS = tm, tP = tm + N, tV = tm + 2 * N, tK = tV + (HD == 128 ? 128 : 64);
    auto head_of = [&](int i) { return head0 + i / nq; };
    auto row_of = [&](int i) { return (first + i % nq) * N; };

    if (warp >= 8) {
        fewer_registers<kOtherRegs>();
        if (warp == 9) {
            // `fixed` tells that the rows behind the sequence are cleared (their weights
            // are 0, 0 times another sequence's NaN is not).
            auto load = [&](const CUtensorMap* m, int i, uint8_t* r, uint64_t* full, uint64_t* empty, uint64_t* fixed, int n_places) {
                const int st = i % n_places;
                uint8_t* dst = r + st * TILE;
                if (!__all_sync(0xffffffffu, i < n_places || bar_wait(empty + st, (i / n_places - 1) & 1, gone))) return false;
                if (lane == 0 && i) {
                    bar_expect(full + st, TILE);
                    load_parts<HD, N>(dst, m, head_of(i), a.heads, (int)t.start + row_of(i), full + st);
                }
                __syncwarp();
                if (ragged && i % nq == nq - 1) {
                    if (!__all_sync(0xffffffffu, bar_wait(full + st, (i / n_places) & 1, gone))) return false;
                    zero_parts<HD, N>(dst, t.len % N);
                    fence_async_smem();
                    __syncwarp();
                }
                if (lane == 0) bar_arrive(fixed + st);
                return true;
            };
            for (int i = 0; i < n; ++i)
                if (!load(&a.q, i, qr, q_full, q_empty, q_fixed, NA) || !load(&a.g, i, gr, g_full, g_empty, g_fixed, NB)) break;
        } else if (warp == 8) {
            if (lane == 0) {
                auto scores = [&](int i) {
                    const int st = i % NA;
                    if (!bar_wait(q_full + st, (i / NA) & 1, gone) || !bar_wait(q_fixed + st, (i / NA) & 1, gone)) return false;
                    parts_rows<HD, N>(tS, smem(ks), smem(qr + st * TILE));
                    commit(s_ready);
                    return true;
                };
                auto dps = [&](int i) {
                    const int st = i % NB;
                    if (!bar_wait(g_full + st, (i / NB) & 1, gone) || !bar_wait(g_fixed + st, (i / NB) & 1, gone)) return false;
                    parts_rows<HD, N>(tP, smem(vs), smem(gr + st * TILE));
                    commit(dp_ready);
                    return true;
                };
                bool ok = bar_wait(kv_full, 0, gone) && scores(0) && bar_wait(kv_full + 1, 0, gone) && dps(0);
                for (int i = 0; ok && i < n; ++i) {
                    const bool more = i + 1 < n;
                    ok = bar_wait(p_ready, i & 1, gone);
                    if (!ok) break;
                    fence_after();
                    parts_weights<HD, N>(tV, tS, smem(gr + (i % NB) * TILE));
                    commit(dv_done);
                    commit(g_empty + i % NB);
                    ok = (!more || scores(i + 1)) && bar_wait(ds_ready, i & 1, gone);
                    if (!ok) break;
                    fence_after();
                    parts_weights<HD, N>(tK, tP, smem(qr + (i % NA) * TILE));
                    commit(dk_done);
                    commit(q_empty + i % NA);
                    ok = !more || dps(i + 1);
                }
            }
            __syncwarp();
        } else if (warp == 10) {
            const long long ks = slot_of(t, t.row0) * a.kv_heads + kvh;
            const float fv = a.fv[ks], vnorm = a.vnorm[ks];
            for (int i = 0; i < n; ++i) {
                const int sl = i & 1, h = head_of(i);
                const bool ok = i < 2 || bar_wait(stat_empty + sl, (i / 2 - 1) & 1, gone);
                if (!__all_sync(0xffffffffu, ok)) break;
                const long long qs = slot_of(t, row_of(i)) * a.heads + h;
                const DsFactors ds = ds_factors(a.fg[qs], a.gnorm[qs], a.dtop[qs], fv, vnorm);
                const float up = ds.up * kPDown;
                if (lane == 0) st_ds[sl] = make_float2(ds.acc, ds.down);
                for (int r = lane; r < N; r += 32) {
                    const int row = row_of(i) + r;
                    float x = INFINITY, d = 0.f;
                    if (row < t.len) {
                        x = a.lse_in[(long long)h * a.tokens + t.start + row];
                        x = x == -INFINITY ? INFINITY : x * kLog2e - kPUp;
                        d = a.delta[(long long)h * a.tokens + t.start + row] * up;
                    }
                    st_lse[sl * N + r] = -x;
                    st_d[sl * N + r] = -d;
                }
                __syncwarp();
                if (lane == 0) bar_arrive(stat_full + sl);
            }
        }
    } else {
        more_registers<kMathRegs>();
        const int half = warp >> 2, row = t.row0 + (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s0 = tS + lanes + C * half, p0 = tP + lanes + C * half;
        // Half the columns of dv and dk each (dim 32: one warpgroup has dv, the other dk).
        constexpr int W = HD == 32 ? 32 : HD / 2;
        const uint32_t v0 = tV + lanes + (HD == 32 ? 0 : W * half), k0 = tK + lanes + (HD == 32 ? 0 : W * half);
        const long long ks = slot_of(t, t.row0) * a.kv_heads + kvh;
        const float fk = a.fk[ks];
        float2 av[W / 2], ak[W / 2];
#pragma unroll
        for (int i = 0; i < W / 2; ++i) av[i] = ak[i] = both(0.f);
        bool ok = true;
        float take_k = 0.f;                // factor of the dK tile that has not been taken yet
        auto add_k = [&](int i) {
            ok = __all_sync(0xffffffffu, bar_wait(dk_done, i & 1, gone));
            if (!ok) return;
            fence_after();
            if (HD == 32) {
                if (half == 1) take32(av, k0, take_k);
            } else {
#pragma unroll
                for (int b = 0; b < W / 32; ++b) take32(ak + 16 * b, k0 + 32 * b, take_k);
            }
            fence_before();
        };
        for (int i = 0; i < n; ++i) {
            const int sl = i & 1, q0 = row_of(i);
            const long long qs = slot_of(t, q0) * a.heads + head_of(i);
            const float fq = a.fq[qs], fg = a.fg[qs], c = score_factor(a.c * fq, fk);
            ok = bar_wait(stat_full + sl, (i / 2) & 1, gone) && bar_wait(s_ready, i & 1, gone);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            const int see = a.causal ? row - q0 - C * half : -1;          // columns from here on see this key
            const bool part = __any_sync(0xffffffffu, see > 0);
            const float* lse = st_lse + sl * N + C * half;
            const float* dd = st_d + sl * N + C * half;
            float2 p[C / 2];
#pragma unroll
            for (int b = 0; b < C / 2; b += 16) {
                uint32_t s[32];
                ld32(s, s0 + 2 * b);
                wait_ld();
#pragma unroll
                for (int x = 0; x < 16; x += 2) {
                    const float4 z = *reinterpret_cast<const float4*>(lse + 2 * (b + x));      // -lse
                    p[b + x] = exp2_both(__ffma2_rn(pair(s[2 * x], s[2 * x + 1]), both(c), make_float2(z.x, z.y)));
                    p[b + x + 1] = exp2_both(__ffma2_rn(pair(s[2 * x + 2], s[2 * x + 3]), both(c), make_float2(z.z, z.w)));
                }
                if (part) {
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        if (2 * (b + x) < see) p[b + x].x = 0.f;
                        if (2 * (b + x) + 1 < see) p[b + x].y = 0.f;
                    }
                }
                put_parts(s0 + 2 * b, p + b);
            }
            wait_st();
            fence_before();
            bar_arrive(p_ready);
            if (i) add_k(i - 1);
            if (!ok) break;
            take_k = fminf(fq * st_ds[sl].y, 3e38f);
            ok = __all_sync(0xffffffffu, bar_wait(dp_ready, i & 1, gone));
            if (!ok) break;
            fence_after();
#pragma unroll
            for (int b = 0; b < C / 2; b += 16) {
                uint32_t s[32];
                ld32(s, p0 + 2 * b);
                wait_ld();
#pragma unroll
                for (int x = 0; x < 16; x += 2) {
                    const float4 z = *reinterpret_cast<const float4*>(dd + 2 * (b + x));       // -D
                    const float2 f = both(st_ds[sl].x);
                    p[b + x] = __fmul2_rn(p[b + x], __ffma2_rn(pair(s[2 * x], s[2 * x + 1]), f, make_float2(z.x, z.y)));
                    p[b + x + 1] = __fmul2_rn(p[b + x + 1], __ffma2_rn(pair(s[2 * x + 2], s[2 * x + 3]), f, make_float2(z.z, z.w)));
                }
                if (part) {
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        if (2 * (b + x) < see) p[b + x].x = 0.f;
                        if (2 * (b + x) + 1 < see) p[b + x].y = 0.f;
                    }
                }
                put_parts(p0 + 2 * b, p + b);
            }
            wait_st();
            fence_before();
            bar_arrive(ds_ready);
            bar_arrive(stat_empty + sl);
            ok = __all_sync(0xffffffffu, bar_wait(dv_done, i & 1, gone));
            if (!ok) break;
            fence_after();
            if (HD != 32 || half == 0) {
#pragma unroll
                for (int b = 0; b < W / 32; ++b) take32(av + 16 * b, v0 + 32 * b, fg * kPDown);
            }
            fence_before();
        }
        if (ok) add_k(n - 1);
        if (ok && row < t.len) {
            if (HD == 32) {
                store32((half ? dk : dv) + row * out_row, av, half ? fabsf(a.scale) : 1.f);
            } else {
#pragma unroll
                for (int b = 0; b < W / 32; ++b) {
                    store32(dv + row * out_row + W * half + 32 * b, av + 16 * b, 1.f);
                    store32(dk + row * out_row + W * half + 32 * b, ak + 16 * b, fabsf(a.scale));
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    settle(gone);
    fence_after();
    if (warp == 8) tmem_free(tm, 512);
    if (threadIdx.x == 0 && *gone) atomicOr(a.err, kErrTcWait);
}

// dq of 128 queries: key tiles pass by.  S has two blocks of columns, dS(j)
// lies in S(j)'s; the order is dP(j+1), dQ(j), S(j+2).
template <int HD>
__device__ __forceinline__ void block_dq(const Args& a, uint8_t* sm, unsigned block, unsigned blocks) {
    using Sh = Shape<HD>;
    using Bs = BwdShape<HD>;
    constexpr int NA = Bs::A, NB = Bs::B, N = Bs::N, TILE = Bs::TILE, C = N / 2;
    uint8_t *qs = sm, *gs = sm + Bs::KEPT, *kr = sm + Bs::RING, *vr = kr + NA * TILE;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Bs::BARS);
    uint64_t *k_full = bars, *k_empty = k_full + NA, *v_full = k_empty + NA, *v_empty = v_full + NB, *fixed = v_empty + NB,
             *qg_full = fixed + 1, *s_ready = qg_full + 2,
             *dp_ready = s_ready + 2, *ds_ready = dp_ready + 1, *dq_done = ds_ready + 1;
    uint32_t* tmem_base = reinterpret_cast<uint32_t*>(dq_done + 1);
    volatile int* gone = reinterpret_cast<volatile int*>(tmem_base + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int head = block % a.heads, kvh = head / a.group;
    const PackedTile t = packed_tile(a.cu, a.n_seqs, a.tokens, kWide, (blocks - 1 - block) / a.heads);
    if (t.row0 >= t.len) return;
    const long long out_row = (long long)a.heads * HD;
    float* dq = a.dq + (t.start * a.heads + head) * HD;
    if (t.seq == a.n_seqs) {
        zero_rows_out(dq, out_row, HD, t.row0, t.len);
        return;
    }
    const int last = a.causal ? min(t.row0 + kWide, t.len) : t.len;
    const int n = (last + N - 1) / N;
    const bool ragged = n * N > t.len;

    if (threadIdx.x == 32 * 9) {
        *gone = 0;
        for (int i = 0; i < NA; ++i) { bar_init(k_full + i, 1); bar_init(k_empty + i, 1); }
        for (int i = 0; i < NB; ++i) { bar_init(v_full + i, 1); bar_init(v_empty + i, 1); }
        bar_init(fixed, 1); bar_init(qg_full, 1); bar_init(qg_full + 1, 1); bar_init(s_ready, 1); bar_init(s_ready + 1, 1);
        bar_init(dp_ready, 1); bar_init(ds_ready, 256); bar_init(dq_done, 1);
        bar_init_done();
        const int r0 = (int)t.start;
        bar_expect(qg_full, Bs::KEPT);
        load_parts<HD, kWide>(qs, &a.q, head, a.heads, r0 + t.row0, qg_full);
        bar_expect(k_full, TILE);
        load_parts<HD, N>(kr, &a.k, kvh, a.kv_heads, r0, k_full);
        bar_expect(qg_full + 1, Bs::KEPT);
        load_parts<HD, kWide>(gs, &a.g, head, a.heads, r0 + t.row0, qg_full + 1);
        bar_expect(v_full, TILE);
        load_parts<HD, N>(vr, &a.v, kvh, a.kv_heads, r0, v_full);
    }
    if (warp == 8) tmem_alloc(tmem_base, 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm = *tmem_base, tS = tm, tP = tm + 2 * N, tQ = tm + 3 * N;

    if (warp >= 8) {
        fewer_registers<kOtherRegs>();
        if (warp == 9) {
            if (lane == 0) {
                const int r0 = (int)t.start;
                for (int j = 1; j < n; ++j) {
                    const int sa = j % NA, sb = j % NB;
                    if (j >= NA && !bar_wait(k_empty + sa, (j / NA - 1) & 1, gone)) break;
                    bar_expect(k_full + sa, TILE);
                    load_parts<HD, N>(kr + sa * TILE, &a.k, kvh, a.kv_heads, r0 + j * N, k_full + sa);
                    if (j >= NB && !bar_wait(v_empty + sb, (j / NB - 1) & 1, gone)) break;
                    bar_expect(v_full + sb, TILE);
                    load_parts<HD, N>(vr + sb * TILE, &a.v, kvh, a.kv_heads, r0 + j * N, v_full + sb);
                }
            }
            __syncwarp();
            if (ragged) {                   // keys behind the sequence: their dS is 0, 0 times NaN would not be
                const int st = (n - 1) % NA;
                if (bar_wait(k_full + st, ((n - 1) / NA) & 1, gone)) {
                    zero_parts<HD, N>(kr + st * TILE, t.len - (n - 1) * N);
                    fence_async_smem();
                }
                __syncwarp();
                if (lane == 0) bar_arrive(fixed);
            }
        } else if (warp == 8) {
            if (lane == 0) {
                auto scores = [&](int j) {
                    if (!bar_wait(k_full + j % NA, (j / NA) & 1, gone)) return false;
                    parts_rows<HD, N>(tS + N * (j & 1), smem(qs), smem(kr + (j % NA) * TILE));
                    commit(s_ready + (j & 1));
                    return true;
                };
                auto dps = [&](int j) {
                    if (!bar_wait(v_full + j % NB, (j / NB) & 1, gone)) return false;
                    parts_rows<HD, N>(tP, smem(gs), smem(vr + (j % NB) * TILE));
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
                    if (ok && ragged && j == n - 1) ok = bar_wait(fixed, 0, gone);
                    if (!ok) break;
                    parts_weights<HD, N>(tQ, tS + N * (j & 1), smem(kr + (j % NA) * TILE));
                    commit(dq_done);
                    commit(k_empty + j % NA);
                    if (j + 2 < n) ok = scores(j + 2);
                }
            }
            __syncwarp();
        }
    } else {
        more_registers<kMathRegs>();
        const int half = warp >> 2, row = t.row0 + (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        constexpr int W = HD == 32 ? 32 : HD / 2;
        const uint32_t q0 = tQ + lanes + (HD == 32 ? 0 : W * half), p0 = tP + lanes + C * half;
        const long long qslot = slot_of(t, t.row0) * a.heads + head;
        const float fq = a.fq[qslot];
        float lse = INFINITY, d = 0.f;
        float2 acc[W / 2];
#pragma unroll
        for (int i = 0; i < W / 2; ++i) acc[i] = both(0.f);
        if (row < t.len) {
            const long long at = (long long)head * a.tokens + t.start + row;
            lse = a.lse_in[at];
            lse = lse == -INFINITY ? INFINITY : lse * kLog2e - kPUp;
            d = a.delta[at];
        }
        bool ok = true;
        float take_f = 0.f;
        auto add_q = [&](int j) {
            ok = __all_sync(0xffffffffu, bar_wait(dq_done, j & 1, gone));
            if (!ok) return;
            fence_after();
            if (HD != 32 || half == 0) {
#pragma unroll
                for (int b = 0; b < W / 32; ++b) take32(acc + 16 * b, q0 + 32 * b, take_f);
            }
            fence_before();
        };
        for (int j = 0; j < n; ++j) {
            const uint32_t s0 = tS + lanes + N * (j & 1) + C * half;
            const long long ks = slot_of(t, j * N) * a.kv_heads + kvh;
            const float c = score_factor(a.c * fq, a.fk[ks]);
            ok = __all_sync(0xffffffffu, bar_wait(s_ready + (j & 1), (j >> 1) & 1, gone));
            if (!ok) break;
            fence_after();
            const int lim = min(t.len, a.causal ? row + 1 : t.len) - j * N - C * half;
            float2 p[C / 2];
#pragma unroll
            for (int b = 0; b < C / 2; b += 16) {
                uint32_t s[32];
                ld32(s, s0 + 2 * b);
                wait_ld();
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    p[b + x] = exp2_both(__ffma2_rn(pair(s[2 * x], s[2 * x + 1]), both(c), both(-lse)));
            }
            if (j) add_q(j - 1);
            if (!ok) break;
            // Read here, not before the weights: registers are what this kernel lacks.
            const DsFactors ds = ds_factors(a.fg[qslot], a.gnorm[qslot], a.dtop[qslot], a.fv[ks], a.vnorm[ks]);
            const float du = d * (ds.up * kPDown);
            take_f = fminf(a.fk[ks] * ds.down, 3e38f);
            ok = __all_sync(0xffffffffu, bar_wait(dp_ready, j & 1, gone));
            if (!ok) break;
            fence_after();
            const bool part = __any_sync(0xffffffffu, lim < C);
#pragma unroll
            for (int b = 0; b < C / 2; b += 16) {
                uint32_t s[32];
                ld32(s, p0 + 2 * b);
                wait_ld();
#pragma unroll
                for (int x = 0; x < 16; ++x)
                    p[b + x] = __fmul2_rn(p[b + x], __ffma2_rn(pair(s[2 * x], s[2 * x + 1]), both(ds.acc), both(-du)));
                if (part) {
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        if (2 * (b + x) >= lim) p[b + x].x = 0.f;
                        if (2 * (b + x) + 1 >= lim) p[b + x].y = 0.f;
                    }
                }
                put_parts(s0 + 2 * b, p + b);
            }
            wait_st();
            fence_before();
            bar_arrive(ds_ready);
        }
        if (ok) add_q(n - 1);
        if (ok && row < t.len && (HD != 32 || half == 0)) {
#pragma unroll
            for (int b = 0; b < W / 32; ++b)
                store32(dq + row * out_row + (HD == 32 ? 0 : W * half) + 32 * b, acc + 16 * b, a.scale);
        }
    }
    fence_before();
    __syncthreads();
    settle(gone);
    fence_after();
    if (warp == 8) tmem_free(tm, 512);
    if (threadIdx.x == 0 && *gone) atomicOr(a.err, kErrTcWait);
}

// One launch for both: the blocks of dq fill the SMs that run out of dk and dv.
template <int HD>
__global__ void __launch_bounds__(kThreads, 1) k_f32_bwd(const __grid_constant__ Args a, unsigned dkv_blocks) {
    extern __shared__ __align__(1024) uint8_t sm[];
    if (blockIdx.x < dkv_blocks) block_dkv<HD>(a, sm, blockIdx.x);
    else block_dq<HD>(a, sm, blockIdx.x - dkv_blocks, gridDim.x - dkv_blocks);
}

// dk and dv of a key/value head from those of its query heads, in their order.
__global__ void __launch_bounds__(256) k_add_heads(const float* __restrict__ dk, const float* __restrict__ dv,
                                                   float* __restrict__ ok, float* __restrict__ ov, int group, int hd,
                                                   long long n) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;         // float4 of an output
    if (i >= n) return;
    const long long row = i / (hd / 4), c = i % (hd / 4);
    for (int t = 0; t < 2; ++t) {
        const float4* in = reinterpret_cast<const float4*>(t ? dv : dk) + row * group * (hd / 4) + c;
        float4 s = in[0];
        for (int g = 1; g < group; ++g) {
            const float4 x = in[(long long)g * (hd / 4)];
            s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
        }
        reinterpret_cast<float4*>(t ? ov : ok)[i] = s;
    }
}

// ── launches ──────────────────────────────────────────────────────────────
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Fewer blocks than twice the SMs leave some idle while others go through a whole
// group: then each query head has a block of its own, for two more tensors of q's
// size.  2048 tokens of 16 heads (4 key/value heads): 64 busy blocks 181 us, 256 of
// them 77 us with the sums.
bool by_head(long long tokens, int heads, int kv_heads) {
    return heads > kv_heads && tokens / kWide * kv_heads < 2 * sm_count();
}

// Workspace: parts of q, k, v (and dO), their factors, what bounds dS, D, and dk and dv by query head.
struct Room {
    __half* parts[4];
    float* factors[4];
    float *vnorm, *gnorm, *dtop, *delta, *dk, *dv;
    size_t bytes;
};
Room room(void* ws, long long tokens, int n_seqs, int heads, int kv_heads, int hd, int backward) {
    const long long slots = packed_slots(tokens, n_seqs, kSplit);
    const int h[4] = {heads, kv_heads, kv_heads, backward ? heads : 0};
    Room r{};
    char* p = static_cast<char*>(ws);
    size_t at = 0;
    for (int i = 0; i < 4; ++i) {
        r.parts[i] = reinterpret_cast<__half*>(p + at);
        at += up256((size_t)tokens * 2 * h[i] * hd * sizeof(__half));
    }
    for (int i = 0; i < 4; ++i) {
        r.factors[i] = reinterpret_cast<float*>(p + at);
        at += up256((size_t)slots * h[i] * sizeof(float));
    }
    if (backward) {
        r.vnorm = reinterpret_cast<float*>(p + at);
        at += up256((size_t)slots * kv_heads * sizeof(float));
        r.gnorm = reinterpret_cast<float*>(p + at);
        at += up256((size_t)slots * heads * sizeof(float));
        r.dtop = reinterpret_cast<float*>(p + at);
        at += up256((size_t)slots * heads * sizeof(float));
        r.delta = reinterpret_cast<float*>(p + at);
        at += up256((size_t)tokens * heads * sizeof(float));
    }
    if (backward && by_head(tokens, heads, kv_heads)) {
        r.dk = reinterpret_cast<float*>(p + at);
        at += up256((size_t)tokens * heads * hd * sizeof(float));
        r.dv = reinterpret_cast<float*>(p + at);
        at += up256((size_t)tokens * heads * hd * sizeof(float));
    }
    r.bytes = at;
    return r;
}

bool parts_map(CUtensorMap* m, const __half* p, long long tokens, int heads, int hd) {
    const int sw = hd * 2 < 128 ? hd * 2 : 128;
    const uint64_t dims[3] = {(uint64_t)hd, (uint64_t)2 * heads, (uint64_t)tokens};
    const uint64_t strides[2] = {(uint64_t)hd * 2, (uint64_t)2 * heads * hd * 2};
    const uint32_t box[3] = {(uint32_t)(sw / 2), 1, (uint32_t)kBoxRows};
    return encode_tensor(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p, dims, strides, box, sw);
}

template <int HD>
int launch(const PackedParams& p, const Room& r, Args& a, bool backward, cudaStream_t s) {
    SplitArgs sp{};
    const Rows in[4] = {p.q, p.k, p.v, p.dout};
    const int h[4] = {p.heads, p.kv_heads, p.kv_heads, backward ? p.heads : 0};
    for (int i = 0; i < 4; ++i) {
        sp.in[i] = in[i]; sp.heads[i] = h[i]; sp.first[i + 1] = sp.first[i] + h[i];
        sp.parts[i] = r.parts[i]; sp.factors[i] = r.factors[i];
    }
    sp.out = static_cast<const float*>(p.out_in); sp.delta = r.delta;
    sp.vnorm = r.vnorm; sp.gnorm = r.gnorm; sp.dtop = r.dtop;
    sp.negate = p.scale < 0.f; sp.cu = p.cu; sp.n_seqs = p.n_seqs; sp.tokens = p.tokens;
    const unsigned slots = (unsigned)packed_slots(p.tokens, p.n_seqs, kSplit);
    k_split<HD><<<slots * sp.first[4], 256, 0, s>>>(sp);
    if (cudaGetLastError() != cudaSuccess) return kErrCuda;
    if (!backward) {
        if (!allow_smem<&k_f32_fwd<HD>>(FwdShape<HD>::SMEM)) return kErrCuda;
        k_f32_fwd<HD><<<slots * p.heads, kThreads, FwdShape<HD>::SMEM, s>>>(a);
        return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
    }
    a.split = by_head(p.tokens, p.heads, p.kv_heads);
    if (a.split) { a.dk = r.dk; a.dv = r.dv; }
    const unsigned dkv_blocks = slots * (a.split ? p.heads : p.kv_heads);
    if (!allow_smem<&k_f32_bwd<HD>>(BwdShape<HD>::SMEM)) return kErrCuda;
    k_f32_bwd<HD><<<dkv_blocks + slots * p.heads, kThreads, BwdShape<HD>::SMEM, s>>>(a, dkv_blocks);
    if (cudaGetLastError() != cudaSuccess) return kErrCuda;
    if (a.split) {
        const long long n = p.tokens * p.kv_heads * (HD / 4);
        k_add_heads<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(r.dk, r.dv, static_cast<float*>(p.dk),
                                                                static_cast<float*>(p.dv), a.group, HD, n);
        if (cudaGetLastError() != cudaSuccess) return kErrCuda;
    }
    return kOk;
}

}  // namespace

size_t attention_packed_f32_workspace(long long tokens, int n_seqs, int heads, int kv_heads, int head_dim, int backward) {
    return room(nullptr, tokens, n_seqs, heads, kv_heads, head_dim, backward).bytes;
}

int attention_packed_f32(const PackedParams& p, int backward, cudaStream_t s) {
    const Room r = room(p.ws, p.tokens, p.n_seqs, p.heads, p.kv_heads, p.head_dim, backward);
    Args a{};
    if (!parts_map(&a.q, r.parts[0], p.tokens, p.heads, p.head_dim) ||
        !parts_map(&a.k, r.parts[1], p.tokens, p.kv_heads, p.head_dim) ||
        !parts_map(&a.v, r.parts[2], p.tokens, p.kv_heads, p.head_dim) ||
        (backward && !parts_map(&a.g, r.parts[3], p.tokens, p.heads, p.head_dim)))
        return kErrUnsupported;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return kErrCuda; }
    a.cu = p.cu; a.n_seqs = p.n_seqs; a.heads = p.heads; a.kv_heads = p.kv_heads; a.group = p.heads / p.kv_heads;
    a.causal = p.causal; a.zero_rest = p.zero_rest; a.tokens = p.tokens;
    a.c = fabsf(p.scale) * kLog2e;
    a.scale = p.scale;
    a.pq = r.parts[0]; a.pk = r.parts[1]; a.pv = r.parts[2]; a.pg = r.parts[3];
    a.fq = r.factors[0]; a.fk = r.factors[1]; a.fv = r.factors[2]; a.fg = r.factors[3];
    a.vnorm = r.vnorm; a.gnorm = r.gnorm; a.dtop = r.dtop;
    a.lse_in = p.lse_in; a.delta = r.delta;
    a.out = static_cast<float*>(p.out); a.lse = p.lse;
    a.dq = static_cast<float*>(p.dq); a.dk = static_cast<float*>(p.dk); a.dv = static_cast<float*>(p.dv);
    a.err = device_error_word(dev);
    if (!a.err) return kErrCuda;
    switch (p.head_dim) {
        case 32: return launch<32>(p, r, a, backward, s);
        case 64: return launch<64>(p, r, a, backward, s);
        default: return launch<128>(p, r, a, backward, s);
    }
}

}  // namespace racb
