// cached_split.cuh -- how the kernels of attention over a paged cache share out
// their work.
//
// Work is split by keys, not by sequences: a unit is some of the rows of one
// (sequence, key/value head), and the key tiles of all units stand in one
// line, cut into equal pieces, one a block, so that caches of any lengths
// keep every SM busy.  Each block reads the lengths and finds its piece; the
// host need not know them.  A unit that lies in one piece is finished there;
// of one that is cut each piece leaves its normalised sum and the logarithm
// (to base 2) of its weight, and k_cached_join joins them; its launch overlaps
// the first kernel.
#pragma once
#include "attn_common.cuh"
#include "tensor_core.cuh"

namespace racb {
namespace {

constexpr int kKeys = 128;                 // keys of a tile

struct Args {
    CachedParams p;
    float c;                               // scale * log2(e)
    int rows;                              // rows of a (sequence, kv head): new rows x heads of the group
    int unit_span, row_units, unit_rows;   // rows from unit to unit; units of a head; rows of a unit
    int start;                             // what a unit's start costs, in tiles: its places on the line before them
    int copies;                            // of the rows in a tile (tensor-core kernel)
    float *part, *part_lse;                // [2 * blocks, unit_rows, dim], [2 * blocks, unit_rows]
    unsigned int* err;
};

__device__ __forceinline__ int rows_in_cache(const CachedParams& p, int b) {
    const long long cap = min((long long)p.table_width * p.page_size, 0x7fff0000LL);
    const long long n = p.lengths[b];
    return (int)(n < 0 ? 0 : (n > cap ? cap : n));
}
__device__ __forceinline__ int new_rows(const CachedParams& p, int b) {
    return p.counts ? max(0, min(p.counts[b], p.nodes)) : p.nodes;
}
// Key tiles of a sequence: one at least, which writes the zeros of an empty one.
__device__ __forceinline__ int tiles_of(const CachedParams& p, int b) {
    return max(1, (rows_in_cache(p, b) + kKeys - 1) / kKeys);
}

// The piece of the line of tiles that a block works on: where it has got to and
// the tiles to go; and the piece's segments, of one unit each.
struct Walk {
    long long left;
    int b, kvh, unit, j;
};
struct Segment {
    int b, kvh, unit, tiles, j0, j1;       // key tiles [j0, j1) of `tiles`
};
// By counting: every role of the kernels steps through the segments, and a 64-bit
// division there is a call that costs the roles' loops their registers.
__device__ __forceinline__ bool next(const Args& a, Walk& w, Segment& s) {
    if (w.left <= 0) return false;
    s.b = w.b;
    s.kvh = w.kvh;
    s.unit = w.unit;
    s.tiles = tiles_of(a.p, w.b);
    s.j0 = w.j;
    s.j1 = (int)min((long long)s.tiles, s.j0 + w.left);
    w.left -= s.j1 - s.j0;
    w.j = s.j1;
    if (w.j == s.tiles) {
        w.j = 0;
        if (++w.unit == a.row_units) {
            w.unit = 0;
            if (++w.kvh == a.p.kv_heads) {
                w.kvh = 0;
                ++w.b;
            }
        }
    }
    return true;
}

// Sum over b < limit of the key tiles, by one warp.
__device__ __forceinline__ long long tiles_before(const CachedParams& p, int limit) {
    long long n = 0;
    for (int b = threadIdx.x & 31; b < limit; b += 32) n += tiles_of(p, b);
#pragma unroll
    for (int off = 16; off; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
    return n;
}

// The beginning of piece i of n, at position total i / n of the line; `left` counts
// the tiles before it.  n: the blocks launched or, where that is less, the positions
// there are.  By one warp: two of them look for a block's two ends at the same time.
__device__ __forceinline__ Walk place(const Args& a, int i, int blocks) {
    const long long per = (long long)a.p.kv_heads * a.row_units;
    const long long total = (tiles_before(a.p, a.p.batch) + (long long)a.p.batch * a.start) * per;
    const long long n_pieces = min((long long)blocks, total);
    const long long pos = i < n_pieces ? total * i / n_pieces : total;
    Walk w{};
    const int lane = threadIdx.x & 31;
    long long at = 0;                      // of sequence w.b: its first position
    w.b = a.p.batch;
    for (int b0 = 0; b0 < a.p.batch; b0 += 32) {
        const bool live = b0 + lane < a.p.batch;
        long long n = live ? tiles_of(a.p, b0 + lane) : 0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, n, off);
            if (lane >= off) n += x;
        }
        // Tiles and positions up to the end of sequence b0 + lane, counted from b0.
        const long long m = n + (long long)a.start * min(lane + 1, a.p.batch - b0);
        const unsigned past = __ballot_sync(0xffffffffu, at + m * per > pos);
        const int l = past ? __ffs(past) - 1 : 32;
        const long long x = __shfl_sync(0xffffffffu, n, l ? l - 1 : 0), y = __shfl_sync(0xffffffffu, m, l ? l - 1 : 0);
        if (l) { w.left += x * per; at += y * per; }
        if (past) { w.b = b0 + l; break; }
    }
    if (w.b == a.p.batch) return w;
    const int n = tiles_of(a.p, w.b);
    const long long u = (pos - at) / (n + a.start);
    w.kvh = (int)u / a.row_units;          // u < per
    w.unit = (int)u % a.row_units;
    w.j = (int)max(0LL, pos - at - u * (n + a.start) - a.start);
    w.left += u * n + w.j;
    return w;
}
// The walk of a block between two such places.
__device__ __forceinline__ Walk between(const Walk (&ends)[2]) {
    Walk w = ends[0];
    w.left = ends[1].left - w.left;
    return w;
}

// Joins the pieces of cut units: a warp a row, eight rows of one unit a block.
template <typename T, int HD>
__global__ void __launch_bounds__(256) k_cached_join(const __grid_constant__ Args a, int launched) {
    const CachedParams& p = a.p;
    const long long per = (long long)p.kv_heads * a.row_units;
    const int parts = (a.unit_rows + 7) / 8, ur = (int)(blockIdx.x % parts) * 8 + (threadIdx.x >> 5);
    const long long bu = blockIdx.x / parts;
    const int b = (int)(bu / per), u = (int)(bu % per);
    const int kvh = u / a.row_units, unit = u % a.row_units, group = p.heads / p.kv_heads;
    const long long total = (tiles_before(p, p.batch) + (long long)p.batch * a.start) * per;
    const int n = tiles_of(p, b);
    const long long blocks = min((long long)launched, total);
    // The unit's places: from t0, its tiles from t1; the blocks of its first and last tile.
    const long long t0 = (tiles_before(p, b) + (long long)b * a.start) * per + (long long)u * (n + a.start), t1 = t0 + a.start;
    const long long c0 = ((t1 + 1) * blocks - 1) / total, c1 = ((t1 + n) * blocks - 1) / total;
    const int cnt = new_rows(p, b), lane = threadIdx.x & 31;
    const long long s0 = 2 * c0 + (total * c0 / blocks >= t0 ? 0 : 1);     // the first piece's place
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (c0 == c1) return;
    const int r = unit * a.unit_span + ur, node = r / group;
    if (ur >= a.unit_rows || r >= a.rows || (node >= cnt && !p.zero_rest)) return;
    float acc[HD / 32], w = 0.f, m = -INFINITY;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) acc[i] = 0.f;
    if (node < cnt) {
        // A running reference point: the pieces are read once.
#pragma unroll 4
        for (long long c = c0; c <= c1; ++c) {
            const long long at = (c == c0 ? s0 : 2 * c) * a.unit_rows + ur;
            const float x = a.part_lse[at], top = fmaxf(m, x), ref = top == -INFINITY ? 0.f : top;
            const float keep = tc::exp2_fast(m - ref), f = tc::exp2_fast(x - ref);
            m = top;
            w = fmaf(w, keep, f);
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) acc[i] = fmaf(f, a.part[at * HD + i * 32 + lane], acc[i] * keep);
        }
    }
    T* out = static_cast<T*>(p.out) + (((long long)b * p.nodes + node) * p.heads + kvh * group + r % group) * HD;
    const float f = w == 0.f ? 0.f : 1.f / w;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) out[i * 32 + lane] = from_f32<T>(acc[i] * f);
}

template <typename T, int HD>
int launch_join(const Args& a, int blocks, cudaStream_t s) {
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((long long)a.p.batch * a.p.kv_heads * a.row_units * ((a.unit_rows + 7) / 8)));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_cached_join<T, HD>, a, blocks) == cudaSuccess ? kOk : kErrCuda;
}

// Rows into units of at most `span`; the pieces' places in the workspace.
inline int fill(Args& a, const CachedParams& p, int span, int blocks) {
    a.p = p;
    // 0 would turn a hidden score's infinity into NaN; 1e-30 weighs the rest alike.
    a.c = p.scale == 0.f ? 1e-30f : p.scale * 1.4426950408889634f;
    a.rows = p.nodes * (p.heads / p.kv_heads);
    a.unit_span = span;
    a.row_units = (a.rows + span - 1) / span;
    a.unit_rows = a.rows < span ? a.rows : span;
    a.part = static_cast<float*>(p.ws);
    a.part_lse = a.part + (size_t)2 * blocks * a.unit_rows * p.head_dim;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return kErrCuda; }
    a.err = device_error_word(dev);
    return a.err ? kOk : kErrCuda;
}
inline size_t pieces_bytes(int blocks, int span, int nodes, int heads, int kv_heads, int head_dim) {
    const long long rows = (long long)nodes * (heads / kv_heads);
    return (size_t)2 * blocks * (rows < span ? rows : span) * (head_dim + 1) * sizeof(float);
}

}  // namespace
}  // namespace racb
