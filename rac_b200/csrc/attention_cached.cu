// attention_cached.cu -- attention of new tokens over a paged key/value cache:
// arguments, the choice of kernels by type, and the float32 kernel.
//
// Sequence b has lengths[b] rows in the cache; the last counts[b] of them are
// new, and queries (b, i, h), i < counts[b], attend over the rows before them
// (all visible) and over the new rows that their mask names: bit j of
// tree[b, i], or j <= i where there is no tree.  One token a sequence is the
// case nodes == 1.  o = sum_j p_j v_j, p = softmax(scale q . k_j) over the
// visible rows; a query that sees no row gives zeros.
//
// float32: a warp takes 32 keys of a tile, the lanes lie along the head, and
// eight rows (new rows x heads of a group) share what is read.  Four keys times
// eight rows are 32 products; adding them up across the lanes by halves leaves
// each lane the score of one (key, row), so that one exp2 a lane weighs all of
// them.  9 instructions for a (key, row) at dim 128 keep eight rows under the
// 44 cycles in which HBM delivers an SM a key; more rows read the cache again
// (from L2, as the units of a head stand side by side in the line of work).
// One token over 300 rows, 32 heads of 128: 16 us a call, the host's time and two launches.
#include "cached_split.cuh"

namespace racb {
namespace {

constexpr int kRowsF32 = 8, kThreadsF32 = 128, kBlocksPerSm = 3;

template <int HD>
__global__ void __launch_bounds__(kThreadsF32, kBlocksPerSm) k_cached_f32(const __grid_constant__ Args a) {
    constexpr int L = HD / 4;              // lanes of a key
    constexpr int G = 32 / L;              // keys of a load
    constexpr int NB = L / 8;              // loads of a batch of four keys
    constexpr int U = 4 / NB;              // batches of a step: four loads
    constexpr int STEPS = 8 / G;           // steps of a warp's 32 keys
    __shared__ float4 so[4][kRowsF32][L];
    __shared__ float2 sml[4][kRowsF32];
    __shared__ Walk ends[2];
    const CachedParams& p = a.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = (lane % L) * 4, group = p.heads / p.kv_heads;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp < 2) {
        const Walk w = place(a, blockIdx.x + warp, gridDim.x);
        if (lane == 0) ends[warp] = w;
    }
    __syncthreads();
    Walk w = between(ends);
    Segment s;
    for (bool first = true; next(a, w, s); first = false) {
        const int len = rows_in_cache(p, s.b), cnt = new_rows(p, s.b), prefix = max(0, len - cnt);
        const float* kp = static_cast<const float*>(p.k.p) + s.kvh * p.k.head + dim;
        const float* vp = static_cast<const float*>(p.v.p) + s.kvh * p.v.head + dim;
        const int* table = p.table + (long long)s.b * p.table_width;
        // Page and slot of this lane's key of a tile; page -1: hidden.
        auto look = [&](int j, int& page, int& slot) {
            const int r = j * kKeys + warp * 32 + lane;
            page = -1;
            slot = 0;
            if (r < len) {
                const int i = r / p.page_size;
                slot = r - i * p.page_size;
                page = table[i];
                if (page < 0 || page >= p.pages) {
                    page = -1;
                    atomicOr(a.err, kErrBadPage);
                }
            }
        };
        int page, slot, page1 = -1, slot1 = 0;
        look(s.j0, page, slot);
        float4 q[kRowsF32], o[kRowsF32];
#pragma unroll
        for (int i = 0; i < kRowsF32; ++i) {
            const int r = s.unit * kRowsF32 + i, node = r / group;
            o[i] = q[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < a.rows) {
                q[i] = *reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + s.b * p.q_batch + node * p.q_node +
                                                        (s.kvh * group + r - node * group) * p.q_head + dim);
                q[i].x *= a.c; q[i].y *= a.c; q[i].z *= a.c; q[i].w *= a.c;
            }
        }
        // This lane's row, and the new rows that it sees.
        const int r = s.unit * kRowsF32 + (lane & 7), node = r / group;
        unsigned long long sees = 0;
        if (r < a.rows) sees = p.tree ? (unsigned long long)p.tree[(long long)s.b * p.nodes + node] : ~0ull >> (63 - node);
        if (len - prefix < 64) sees &= (1ull << (len - prefix)) - 1;
        float m = -INFINITY, l = 0.f;

        auto fetch = [&](int step, int pg, int sl, float4 (&k)[4], float4 (&v)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = (step * 4 + i) * G + lane / L;
                const long long x = __shfl_sync(0xffffffffu, pg, key), y = __shfl_sync(0xffffffffu, sl, key);
                k[i] = v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (x >= 0) {
                    k[i] = __ldg(reinterpret_cast<const float4*>(kp + x * p.k.page + y * p.k.row));
                    v[i] = __ldg(reinterpret_cast<const float4*>(vp + x * p.v.page + y * p.v.row));
                }
            }
        };
        float4 k[4], v[4], k1[4], v1[4];
        fetch(0, page, slot, k, v);
        for (int j = s.j0; j < s.j1; ++j) {
            if (j + 1 < s.j1) look(j + 1, page1, slot1);
            const unsigned live = __ballot_sync(0xffffffffu, page >= 0);
#pragma unroll 1
            for (int step = 0; step < STEPS; ++step) {
                if (step + 1 < STEPS) fetch(step + 1, page, slot, k1, v1);
                else if (j + 1 < s.j1) fetch(0, page1, slot1, k1, v1);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float d[L];
#pragma unroll
                    for (int i = 0; i < NB; ++i)
#pragma unroll
                        for (int x = 0; x < kRowsF32; ++x) {
                            const float4 kk = k[u * NB + i];
                            const float2 h = __ffma2_rn(make_float2(q[x].x, q[x].y), make_float2(kk.x, kk.y),
                                                        __fmul2_rn(make_float2(q[x].z, q[x].w), make_float2(kk.z, kk.w)));
                            d[i * 8 + x] = h.x + h.y;
                        }
                    // Sums over the L lanes by halves: lane i ends with product i % L.
#pragma unroll
                    for (int off = L / 2; off; off >>= 1) {
                        const bool up = lane & off;
#pragma unroll
                        for (int i = 0; i < off; ++i) {
                            const float send = up ? d[i] : d[i + off], keep = up ? d[i + off] : d[i];
                            d[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
                        }
                    }
                    const int key = (step * 4 + u * NB + ((lane % L) >> 3)) * G + lane / L;
                    const int rel = j * kKeys + warp * 32 + key - prefix;
                    const bool see = (live >> key & 1) && (rel < 0 || (rel < 64 && (sees >> rel & 1)));
                    const float x = see ? d[0] : -INFINITY;
                    float top = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    // The reference point moves only when a weight would pass 2^8.
                    if (__any_sync(0xffffffffu, top > m + 8.f)) {
                        const float f = top > m + 8.f ? exp2f(m - top) : 1.f;
                        if (top > m + 8.f) m = top;
                        l *= f;
#pragma unroll
                        for (int i = 0; i < kRowsF32; ++i) {
                            const float y = __shfl_sync(0xffffffffu, f, i);
                            o[i].x *= y; o[i].y *= y; o[i].z *= y; o[i].w *= y;
                        }
                    }
                    // No maximum yet: the score is minus infinity, or NaN, which maxima pass over.
                    const float wgt = !see ? 0.f : m != -INFINITY ? exp2f(x - m) : x == -INFINITY ? 0.f : x;
                    l += wgt;
#pragma unroll
                    for (int i = 0; i < NB; ++i)
#pragma unroll
                        for (int y = 0; y < kRowsF32; ++y) {
                            const float z = __shfl_sync(0xffffffffu, wgt, (lane & ~(L - 1)) | (i * 8 + y));
                            const float4 vv = v[u * NB + i];
                            const float2 lo = __ffma2_rn(make_float2(z, z), make_float2(vv.x, vv.y), make_float2(o[y].x, o[y].y));
                            const float2 hi = __ffma2_rn(make_float2(z, z), make_float2(vv.z, vv.w), make_float2(o[y].z, o[y].w));
                            o[y] = make_float4(lo.x, lo.y, hi.x, hi.y);
                        }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) { k[i] = k1[i]; v[i] = v1[i]; }
            }
            page = page1;
            slot = slot1;
        }
        // The key groups of a warp, then the warps.
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
#pragma unroll
        for (int i = 0; i < kRowsF32; ++i) {
#pragma unroll
            for (int off = L; off < 32; off <<= 1) {
                o[i].x += __shfl_xor_sync(0xffffffffu, o[i].x, off);
                o[i].y += __shfl_xor_sync(0xffffffffu, o[i].y, off);
                o[i].z += __shfl_xor_sync(0xffffffffu, o[i].z, off);
                o[i].w += __shfl_xor_sync(0xffffffffu, o[i].w, off);
            }
            if (lane < L) so[warp][i][lane] = o[i];
        }
        if (lane < kRowsF32) sml[warp][lane] = make_float2(m, l);
        __syncthreads();
        const bool whole = s.j1 - s.j0 == s.tiles;
        const long long piece_at = 2LL * blockIdx.x + (first ? 0 : 1);
        for (int e = threadIdx.x; e < kRowsF32 * L; e += kThreadsF32) {
            const int ur = e / L, c = e % L, row = s.unit * kRowsF32 + ur, nd = row / group;
            if (ur >= a.unit_rows || row >= a.rows) continue;
            float M = -INFINITY, W = 0.f;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 4; ++i) M = fmaxf(M, sml[i][ur].x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 z = sml[i][ur];
                const float f = z.x == -INFINITY ? 0.f : exp2f(z.x - M);
                const float4 x = so[i][ur][c];
                W = fmaf(f, z.y, W);
                y.x = fmaf(f, x.x, y.x); y.y = fmaf(f, x.y, y.y); y.z = fmaf(f, x.z, y.z); y.w = fmaf(f, x.w, y.w);
            }
            const bool mine = nd < cnt;
            const float inv = W == 0.f || !mine ? 0.f : 1.f / W;
            y = inv == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
            if (whole) {
                if (mine || p.zero_rest)
                    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + (((long long)s.b * p.nodes + nd) * p.heads +
                                                                             s.kvh * group + row - nd * group) * HD + c * 4) = y;
            } else if (mine) {
                *reinterpret_cast<float4*>(a.part + (piece_at * a.unit_rows + ur) * HD + c * 4) = y;
                if (c == 0) a.part_lse[piece_at * a.unit_rows + ur] = W == 0.f ? -INFINITY : M + log2f(W);
            }
        }
        __syncthreads();
    }
}

template <int HD>
int launch_f32(const Args& a, int blocks, cudaStream_t s) {
    k_cached_f32<HD><<<blocks, kThreadsF32, 0, s>>>(a);
    if (cudaGetLastError() != cudaSuccess) return kErrCuda;
    return launch_join<float, HD>(a, blocks, s);
}

int cached_f32(const CachedParams& p, int blocks, cudaStream_t s) {
    Args a{};
    if (int st = fill(a, p, kRowsF32, blocks)) return st;
    switch (p.head_dim) {
        case 32: return launch_f32<32>(a, blocks, s);
        case 64: return launch_f32<64>(a, blocks, s);
        default: return launch_f32<128>(a, blocks, s);
    }
}

}  // namespace

// Two pieces a block, of the kernel that needs more.
size_t attention_cached_workspace(int, int nodes, int heads, int kv_heads, int head_dim) {
    const int sms = sm_count();
    const size_t x = attention_cached_tc_workspace(sms, nodes, heads, kv_heads, head_dim),
                 y = pieces_bytes(kBlocksPerSm * sms, kRowsF32, nodes, heads, kv_heads, head_dim);
    return x > y ? x : y;
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
    if ((long long)p.batch * p.kv_heads * ((long long)p.nodes * (p.heads / p.kv_heads)) >= (1LL << 31) ||
        p.heads / p.kv_heads > 4096)
        return kErrInvalidDim;
    const int sms = sm_count();
    if (!p.ws || (reinterpret_cast<uintptr_t>(p.ws) & 15u) ||
        p.ws_bytes < attention_cached_workspace(p.batch, p.nodes, p.heads, p.kv_heads, p.head_dim))
        return kErrAlloc;
    return p.type == kF32 ? cached_f32(p, kBlocksPerSm * sms, s) : attention_cached_tc(p, sms, s);
}

}  // namespace racb
