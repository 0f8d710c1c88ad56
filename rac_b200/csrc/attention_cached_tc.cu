// attention_cached_tc.cu -- attention of new tokens over a paged cache on the
// tensor cores, float16 and bfloat16.
//
// The rows of one product are the new rows of a sequence times the query heads
// of one key/value head: 4 for a single token with a group of 4, up to 256 for
// a tree, in one or two tiles of 128 (rows that do not exist cost matrix time,
// but the cache's bytes bound this kernel: 128 keys are 64 KB at dim 128, some
// 2800 cycles of an SM's share of HBM, against 1024 of a tile's two products).
// Up to 32 (64) rows stand in the tile four times (twice), and each copy weighs
// a quarter (half) of a tile's keys: the four warps that read a tile's lanes
// share its softmax, which one warp alone would take 3000 cycles for.
// Keys and values come through the page table by 16-byte asynchronous copies,
// four warps of them, into a ring; hidden rows and bad pages become zeros on
// the way, and their scores are masked by bits that the loading warps note.
// (TMA boxes for pages of 16 rows and more: 1 % faster, not worth a second way.)
// With two row tiles each has its own issuing thread; one thread for both spent
// 2 x 500 cycles a tile on the way between them.
// Measured, bf16, dim 128, 32 heads on 8: one token for each of 64 sequences of 500
// to 8100 rows 243 us, 4.7 TB/s of the cache's bytes, bound by them and by each
// block's way to its first tile; 48 tree nodes for each of 8 sequences of 777 to
// 16384 rows 121 us, bound by the exponentials of both row tiles and, 16 us, the join.
#include "cached_split.cuh"

namespace racb {
namespace {

using namespace tc;

constexpr int kRowTile = 128, kUnitRows = 256;
// Warps 0-3, 4-7: softmax of row tile 0, 1; 8-11: loads; 12, 13: matrix instructions of row tile 0, 1;
// 14, 15 fill the warpgroup.
constexpr int kThreads = 512;
// Up to 64 rows, which stand in the one tile several times; up to 128; up to 256 in two tiles.
// One kernel for the first and the others took 235 us for 64 single tokens and 154 for
// trees, where kernels apart took 220 and 136: the registers of one are not those of the other.
enum Rows { kCopies, kOneTile, kTwoTiles };
// Registers: a softmax thread holds its row's 128 scores, with copies a half or a quarter of them.
template <Rows ROWS>
struct Regs {
    static constexpr bool MANY = ROWS != kCopies;
    static constexpr int LAUNCH = 128, MATH = MANY ? 184 : 160, LOAD = MANY ? 80 : 104, OTHER = MANY ? 64 : 88;
    static_assert(MATH * 256 + LOAD * 128 + OTHER * 128 <= LAUNCH * kThreads, "register split");
};
constexpr int kTurnCycles = 4000;          // that the second row tile's softmax lets the first go ahead, at most
constexpr int kInfo = 8;                   // tiles of key masks in flight

template <int HD>
struct Shape {
    static constexpr int SW = HD * 2 < 128 ? HD * 2 : 128;
    static constexpr int BOXES = HD * 2 / SW;
    static constexpr int BOX = kKeys * SW;
    static constexpr int TILE = BOXES * BOX;
    static constexpr int STAGES = HD == 128 ? 4 : HD == 64 ? 8 : 12;
    static constexpr int RING = 2 * TILE, OFFS = RING + STAGES * TILE;
    static constexpr int OKS = OFFS + 2 * 2 * kKeys * 8, BARS = OKS + kInfo * 16;
    static constexpr int WALK = BARS + 512, JOIN = WALK + 128;      // JOIN, twice: [128][17] floats, [128] float2
    static constexpr int JOIN1 = kRowTile * 17 * 4 + kRowTile * 8, SMEM = JOIN + 2 * JOIN1;
    static constexpr int CH = HD / 8;                               // 16-byte units of a row
};
static_assert(Shape<128>::SMEM <= 227 * 1024, "shared memory");

// Byte offset of 16-byte unit c of row r in a swizzled tile.
template <int HD>
__device__ __forceinline__ uint32_t place(int r, int c) {
    using Sh = Shape<HD>;
    constexpr int U = Sh::SW / 16;
    const int sw = U == 8 ? r & 7 : (r >> 1) & 3;
    return (c / U) * Sh::BOX + r * Sh::SW + (((c % U) ^ sw) << 4);
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
// The barrier gets this thread's arrival once its copies so far have landed.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem(bar)) : "memory");
}
// A barrier of 128 threads that gives up like every other wait.
__device__ __forceinline__ bool group_sync(uint64_t* bar, uint32_t& phase, volatile int* gone) {
    bar_arrive(bar);
    const bool ok = bar_wait(bar, phase & 1, gone);
    ++phase;
    return __all_sync(0xffffffffu, ok);
}

// Scores that are not visible (bits of `see`) become the least there are.
__device__ __forceinline__ void hide_scores(uint32_t (&v)[32], uint32_t see, bool neg) {
    const uint32_t hide = neg ? 0x7f800000u : 0xff800000u;
#pragma unroll
    for (int i = 0; i < 32; ++i)
        if (!(see >> i & 1)) v[i] = hide;
}
// Scores of 32 keys (columns at ts + 32 b of the thread's row).
__device__ __forceinline__ void load_scores(uint32_t (&v)[32], uint32_t ts, int b, bool part, uint32_t see, bool neg) {
    ld32(v, ts + 32 * b);
    wait_ld();
    if (part) hide_scores(v, see, neg);
}
__device__ __forceinline__ float largest(const uint32_t (&v)[32], bool neg) { return neg ? smallest32(v) : largest32(v); }
// Weights exp2(c s - ref) of 32 keys, packed to ts + 16 b; returns their sum.
template <typename T>
__device__ __forceinline__ float put_weights(const uint32_t (&v)[32], uint32_t ts, int b, float c, float ref) {
    uint32_t q[16];
    float2 add[2] = {both(0.f), both(0.f)};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float2 e = exp2_both(__ffma2_rn(pair(v[2 * i], v[2 * i + 1]), both(c), both(-ref)));
        add[i & 1] = __fadd2_rn(add[i & 1], e);
        q[i] = pack2<T>(e.x, e.y);
    }
    st16(ts + 16 * b, q);
    return (add[0].x + add[0].y) + (add[1].x + add[1].y);
}

template <typename T, int HD, Rows ROWS>
__global__ void __launch_bounds__(kThreads, 1) k_cached_tc(const __grid_constant__ Args a) {
    using Sh = Shape<HD>;
    // Two row tiles: each has a block of S columns and a thread that issues its
    // products, and they take turns.  One: it has both blocks, and tile g's scores
    // lie in block g & 1.
    constexpr int ST = Sh::STAGES, NW = ROWS == kTwoTiles ? 2 : 1;
    constexpr bool MANY = ROWS != kCopies;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint8_t *qs = sm, *ring = sm + Sh::RING;
    long long* offs = reinterpret_cast<long long*>(sm + Sh::OFFS);         // [2][k, v][128]
    uint32_t* oks = reinterpret_cast<uint32_t*>(sm + Sh::OKS);             // [kInfo][4]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Sh::BARS);
    uint64_t *full = bars, *empty = full + ST, *info = empty + ST, *q_full = info + kInfo, *q_empty = q_full + 2,
             *s_ready = q_empty + 2, *p_ready = s_ready + 2, *o_ready = p_ready + 2, *pv_done = o_ready + 2,
             *load_sync = pv_done + 1, *math_sync = load_sync + 1;   // math_sync: two
    uint32_t* tmem_base = reinterpret_cast<uint32_t*>(math_sync + 2);
    volatile int *gone = reinterpret_cast<volatile int*>(tmem_base + 1), *weighed = gone + 1;
    Walk(&ends)[2] = *reinterpret_cast<Walk(*)[2]>(sm + Sh::WALK);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const CachedParams& p = a.p;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        *gone = 0;
        *weighed = 0;
        for (int i = 0; i < ST; ++i) { bar_init(full + i, 128); bar_init(empty + i, NW); }
        for (int i = 0; i < kInfo; ++i) bar_init(info + i, 4);
        for (int i = 0; i < 2; ++i) {
            bar_init(q_full + i, 128); bar_init(q_empty + i, NW); bar_init(s_ready + i, 1); bar_init(p_ready + i, 128);
            bar_init(o_ready + i, 1);
        }
        bar_init(pv_done, 1);
        bar_init(load_sync, 128);
        bar_init(math_sync, 128);
        bar_init(math_sync + 1, 128);
        bar_init_done();
    }
    if (warp == 12) tmem_alloc(tmem_base, 512);
    if (warp == 8 || warp == 9) {
        const Walk w = place(a, blockIdx.x + warp - 8, gridDim.x);
        if (lane == 0) ends[warp - 8] = w;
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tm = *tmem_base, tS = tm, tO = tm + 256;
    Walk w = between(ends);
    Segment s;

    if (warp >= 12) {
        fewer_registers<Regs<ROWS>::OTHER>();
        const int x = warp - 12;           // row tile
        if (x < NW && lane == 0) {
            constexpr uint32_t iqk = instruction<T>(kRowTile, kKeys, false), ipv = instruction<T>(kRowTile, HD, true);
            int g = 0, seg = 0;            // tiles and segments so far
            bool ok = true, more = next(a, w, s);
            Segment later = s;
            while (ok && more) {
                const int n = s.j1 - s.j0, qslot = NW == 1 ? seg & 1 : 0;
                auto landed = [&](int e) {                     // entry e of the ring: keys, then values of a tile
                    if (!bar_wait(full + e % ST, (e / ST) & 1, gone)) return false;
                    fence_async_smem();    // the copies' writes, for the matrix instructions
                    return true;
                };
                auto scores = [&](int j) {                     // key tile j of the segment
                    const int e = 2 * (g + j), buf = NW == 2 ? x : (g + j) & 1;
                    if (!landed(e)) return false;
                    product_ss<HD / 16, Sh::SW>(tS + buf * kKeys, smem(qs + (NW == 1 ? qslot : x) * Sh::TILE),
                                                smem(ring + (e % ST) * Sh::TILE), Sh::BOX, iqk);
                    commit(s_ready + buf);
                    commit(empty + e % ST);
                    if (j == n - 1) commit(q_empty + qslot);
                    return true;
                };
                ok = bar_wait(q_full + qslot, (NW == 1 ? seg >> 1 : seg) & 1, gone);
                if (!ok) break;
                ok = scores(0);
                if (ok && NW == 1 && n > 1) ok = scores(1);
                for (int j = 0; ok && j < n; ++j) {
                    // Weights of two tiles may be ready before the values of the first have
                    // landed: a barrier for each block of S columns.
                    const int e = 2 * (g + j) + 1, buf = NW == 2 ? x : (g + j) & 1;
                    ok = landed(e) && bar_wait(p_ready + buf, (NW == 2 ? g + j : (g + j) >> 1) & 1, gone);
                    if (!ok) break;
                    fence_after();
                    const uint64_t vb = operand<Sh::SW>(smem(ring + (e % ST) * Sh::TILE), Sh::BOX, 8 * Sh::SW);
                    const uint32_t pw = tS + buf * kKeys;
#pragma unroll
                    for (int k = 0; k < kKeys; k += 16)
                        mma_ts(tO + (NW == 2 ? x : seg & 1) * 128, pw + k / 2, vb + (k * Sh::SW >> 4), ipv, j > 0 || k > 0);
                    if (NW == 1) commit(pv_done);
                    commit(empty + e % ST);
                    if (j == n - 1) commit(o_ready + (NW == 2 ? x : seg & 1));
                    else if (NW == 2) ok = scores(j + 1);
                    else if (j + 2 < n) ok = scores(j + 2);
                    if (j == 0) more = next(a, w, later);
                }
                g += n;
                ++seg;
                s = later;
            }
        }
        __syncwarp();
    } else if (warp >= 8) {
        fewer_registers<Regs<ROWS>::LOAD>();
        const int tid = threadIdx.x - 256;
        const char *kp = static_cast<const char*>(p.k.p), *vp = static_cast<const char*>(p.v.p);
        // A thread copies unit c of rows row0, row0 + STEP, ...; STEP is a multiple of 8,
        // so that the swizzle is the same for all of them.
        constexpr int STEP = 128 / Sh::CH, N = kKeys / STEP;
        static_assert(STEP % 8 == 0, "swizzle");
        const int c = tid % Sh::CH, row0 = tid / Sh::CH;
        const uint32_t dst0 = smem(ring) + place<HD>(row0, c);
        const int group = p.heads / p.kv_heads, span = MANY ? kRowTile : kRowTile / a.copies;
        const float per_group = 1.f / group;
        int e = 0, g = 0, seg = 0;                             // ring entries, tiles, segments so far
        uint32_t syncs = 0;
        bool ok = true, more = next(a, w, s);
        // The next segment and its first page are looked up while the first tile of
        // this one is under way: each lookup is a trip to memory that is busy.
        Segment later = s;
        int later_page = -1;
        auto page_of = [&](const Segment& x, int j) {
            const int r = j * kKeys + tid;
            return r < rows_in_cache(p, x.b) ? p.table[(long long)x.b * p.table_width + r / p.page_size] : -1;
        };
        int page = more ? page_of(s, s.j0) : -1;
        while (ok && more) {
            const int len = rows_in_cache(p, s.b);
            for (int j = s.j0; j < s.j1; ++j, ++g) {
                const int r = j * kKeys + tid;
                const bool live = page >= 0 && page < p.pages;
                if (!live && r < len) atomicOr(a.err, kErrBadPage);
                const int slot = r % p.page_size;
                long long* o = offs + (g & 1) * 2 * kKeys;
                o[tid] = live ? (page * p.k.page + s.kvh * p.k.head + slot * p.k.row) * (long long)sizeof(T) : -1;
                o[kKeys + tid] = live ? (page * p.v.page + s.kvh * p.v.head + slot * p.v.row) * (long long)sizeof(T) : -1;
                const uint32_t bits = __ballot_sync(0xffffffffu, live);
                if (lane == 0) {
                    oks[(g % kInfo) * 4 + warp - 8] = bits;
                    bar_arrive(info + g % kInfo);
                }
                if (j + 1 < s.j1) page = page_of(s, j + 1);
                ok = group_sync(load_sync, syncs, gone);
                for (int kv = 0; kv < 2; ++kv, ++e) {
                    if (e >= ST && ok) ok = bar_wait(empty + e % ST, (e / ST - 1) & 1, gone);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const uint32_t dst = dst0 + (e % ST) * Sh::TILE;
                    const char* src = (kv ? vp : kp) + c * 16;
                    const long long* at = o + kv * kKeys + row0;
#pragma unroll
                    for (int i0 = 0; i0 < N; i0 += 8) {
                        long long x[8];
#pragma unroll
                        for (int i = 0; i < 8 && i0 + i < N; ++i) x[i] = at[(i0 + i) * STEP];
#pragma unroll
                        for (int i = 0; i < 8 && i0 + i < N; ++i)
                            copy16(dst + (i0 + i) * STEP * Sh::SW, x[i] < 0 ? static_cast<const char*>(p.q) : src + x[i],
                                   x[i] >= 0);
                    }
                    copies_arrive(full + e % ST);
                }
                if (!ok) break;
                if (j == s.j0) {
                    // Behind the first keys and values: their room comes free before the queries' does.
                    const int qslot = NW == 1 ? seg & 1 : 0, use = NW == 1 ? seg >> 1 : seg;
                    if (use > 0) ok = bar_wait(q_empty + qslot, (use - 1) & 1, gone);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    // Queries: row r of the unit is new row r / group, head r % group of the group.
                    const int r0 = s.unit * kUnitRows;
                    const uint32_t qdst = smem(qs) + (NW == 1 ? qslot : 0) * Sh::TILE + place<HD>(row0, c);
                    const T* q = static_cast<const T*>(p.q) + s.b * p.q_batch + s.kvh * group * p.q_head + c * 8;
                    for (int x = 0; x < NW; ++x) {
#pragma unroll 4
                        for (int i = 0; i < N; ++i) {
                            const int pr = row0 + i * STEP, r = NW == 2 ? x * kRowTile + pr : pr & (span - 1);
                            const bool live = r < a.unit_rows && r0 + r < a.rows;
                            // (r0 + r) / group: a half is further from every quotient than float rounding reaches.
                            const int node = (int)((r0 + r + 0.5f) * per_group), h = (r0 + r) - node * group;
                            copy16(qdst + x * Sh::TILE + i * STEP * Sh::SW, live ? q + node * p.q_node + h * p.q_head : static_cast<const T*>(p.q),
                                   live);
                        }
                    }
                    copies_arrive(q_full + qslot);
                    more = next(a, w, later);
                    if (more) later_page = page_of(later, later.j0);
                }
            }
            s = later;
            page = later_page;
            ++seg;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        more_registers<Regs<ROWS>::MATH>();
        const int x = warp >> 2, group = p.heads / p.kv_heads, span = MANY ? kRowTile : kRowTile / a.copies;
        const int lane_row = (warp & 3) * 32 + lane, copy = lane_row / span, row = lane_row & (span - 1);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        float* join = reinterpret_cast<float*>(sm + Sh::JOIN + x * Sh::JOIN1);
        float2* join_ml = reinterpret_cast<float2*>(join + kRowTile * 17);
        const bool neg = a.c < 0.f;
        int g = 0, seg = 0;
        uint32_t syncs = 0;
        bool ok = true;
        while (ok && next(a, w, s)) {
            const int n = s.j1 - s.j0;
            if (NW == 1) {
                // One row tile: the warpgroups take turns by segment, and one stores its
                // sums while the other weighs the next segment's scores.
                if ((seg & 1) != x) { g += n; ++seg; continue; }
                // Up to here the barriers below have been another's to wait for.
                if (seg) ok = __all_sync(0xffffffffu, bar_wait(o_ready + ((seg - 1) & 1), ((seg - 1) >> 1) & 1, gone));
                if (!ok) break;
            }
            const uint32_t to = tm + lanes + 256 + x * 128;
            const int ur = (NW == 2 ? x * kRowTile : 0) + row, r = s.unit * kUnitRows + ur;   // row of the unit, of the head
            const bool mine = ur < a.unit_rows && r < a.rows;
            const int cnt = new_rows(p, s.b), len = rows_in_cache(p, s.b), node = r / group;
            const bool busy = __any_sync(0xffffffffu, mine);                              // else nothing to weigh
            const int prefix = max(0, len - cnt);
            unsigned long long sees = 0;
            if (mine) sees = p.tree ? (unsigned long long)p.tree[(long long)s.b * p.nodes + node] : ~0ull >> (63 - node);
            if (len - prefix < 64) sees &= (1ull << (len - prefix)) - 1;
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < n; ++j) {
                const int t = g + j, buf = NW == 2 ? x : t & 1;
                ok = bar_wait(s_ready + buf, (NW == 2 ? t : t >> 1) & 1, gone) &&
                     bar_wait(info + t % kInfo, (t / kInfo) & 1, gone);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                fence_after();
                if (NW == 2 && x == 1 && busy) {
                    // After the first row tile's weights, so that one's products run under the
                    // other's exponentials; in step both take 2900 cycles instead of 2000 (119.4
                    // us for the trees, 115.5 in turn).  Only a matter of pace: nothing depends on it.
                    for (const long long t0 = clock64(); *weighed <= t && clock64() - t0 < kTurnCycles;) {}
                    __syncwarp();
                }
                if (busy) {
                    const uint32_t ts = tm + lanes + buf * kKeys;
                    const uint32_t* in = oks + (t % kInfo) * 4;
                    const int pre = prefix - (s.j0 + j) * kKeys;       // keys of the prefix in this tile
                    const bool part = pre < kKeys || (in[0] & in[1] & in[2] & in[3]) != 0xffffffffu;
                    // Visible: keys below pre, then the row's own mask, whose bit 0 stands at `at`.
                    auto visible = [&](int b) {
                        const int at = pre - 32 * b;
                        uint32_t see = 0;
                        if (at >= 32) see = 0xffffffffu;
                        else if (at >= 0) see = (uint32_t)(sees << at) | ((1u << at) - 1);
                        else if (at > -64) see = (uint32_t)(sees >> -at);
                        return see & in[b];
                    };
                    // The reference point moves only when a weight would pass 2^8.
                    auto move = [&](float top) {
                        if (j == 0) {
                            m = top;
                        } else if (__any_sync(0xffffffffu, top > m + 8.f)) {
                            const float up = top > m + 8.f ? exp2_fast(m - top) : 1.f;
                            if (top > m + 8.f) m = top;
                            l *= up;
                            if (NW == 1) { // the last product may still run; with two tiles S has waited for it
                                ok = __all_sync(0xffffffffu, bar_wait(pv_done, (t - 1) & 1, gone));
                                fence_after();
                            }
#pragma unroll 1
                            for (int b = 0; b < HD / 32; ++b) {
                                uint32_t o[32];
                                ld32(o, to + 32 * b);
                                wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * up);
                                st32(to + 32 * b, o);
                            }
                        }
                        return m == -INFINITY ? 0.f : m;
                    };
                    const uint32_t none[16] = {};
                    if (!MANY && a.copies == 4) {      // this copy's 32 keys; the others weigh the rest
                        uint32_t v[32];
                        load_scores(v, ts, copy, part, visible(copy), neg);
                        const float ref = move(largest(v, neg) * a.c);
#pragma unroll
                        for (int b = 0; b < 4; ++b)
                            if (b != copy) st16(ts + 16 * b, none);
                        l += put_weights<T>(v, ts, copy, a.c, ref);
                    } else if (!MANY) {
                        uint32_t v[2][32];
                        const int b0 = 2 * copy;
                        load_scores(v[0], ts, b0, part, visible(b0), neg);
                        load_scores(v[1], ts, b0 + 1, part, visible(b0 + 1), neg);
                        const float y0 = largest(v[0], neg), y1 = largest(v[1], neg);
                        const float ref = move((neg ? fminf(y0, y1) : fmaxf(y0, y1)) * a.c);
                        st16(ts + 32 - 16 * b0, none);
                        st16(ts + 48 - 16 * b0, none);
                        l += put_weights<T>(v[0], ts, b0, a.c, ref);
                        l += put_weights<T>(v[1], ts, b0 + 1, a.c, ref);
                    } else {
                        uint32_t v[4][32];
#pragma unroll
                        for (int b = 0; b < 4; ++b) ld32(v[b], ts + 32 * b);
                        wait_ld();
                        if (part) {
#pragma unroll
                            for (int b = 0; b < 4; ++b) hide_scores(v[b], visible(b), neg);
                        }
                        float y[4];
#pragma unroll
                        for (int b = 0; b < 4; ++b) y[b] = largest(v[b], neg);
                        const float ref = move((neg ? fminf(fminf(y[0], y[1]), fminf(y[2], y[3]))
                                                    : fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]))) * a.c);
#pragma unroll
                        for (int b = 0; b < 4; ++b) l += put_weights<T>(v[b], ts, b, a.c, ref);
                    }
                    if (!ok) break;
                    wait_st();
                }
                fence_before();
                bar_arrive(p_ready + buf);
                if (NW == 2 && threadIdx.x == 0) *weighed = t + 1;
            }
            if (ok) ok = __all_sync(0xffffffffu, bar_wait(o_ready + x, (NW == 2 ? seg : seg >> 1) & 1, gone));
            if (!ok) break;
            fence_after();
            const bool whole = n == s.tiles, live = mine && node < cnt;
            const long long piece_at = 2LL * blockIdx.x + (seg ? 1 : 0);
            T* out = static_cast<T*>(p.out) +
                     (((long long)s.b * p.nodes + node) * p.heads + s.kvh * group + r % group) * HD;
            float* part = a.part + (piece_at * a.unit_rows + ur) * HD;
            // Four sums of the row, normalised: to the output where the unit is whole.
            auto store4 = [&](int at, const float (&f)[4]) {
                if (whole) {
                    if (mine && (live || p.zero_rest))
                        *reinterpret_cast<uint2*>(out + at) =
                            live ? make_uint2(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3])) : make_uint2(0u, 0u);
                } else if (live) {
                    *reinterpret_cast<float4*>(part + at) = make_float4(f[0], f[1], f[2], f[3]);
                }
            };
            if (!MANY) {
                // The copies' sums of a row become one: each with its own reference point.
                join_ml[lane_row] = make_float2(m, l);
                ok = group_sync(math_sync + x, syncs, gone);
                float M = -INFINITY, L = 0.f;
                for (int i = row; i < kRowTile; i += span) M = fmaxf(M, join_ml[i].x);
                for (int i = row; i < kRowTile; i += span) {
                    const float2 y = join_ml[i];
                    L += y.x == -INFINITY ? y.y : y.y * exp2_fast(y.x - M);      // without a maximum: 0, or NaN
                }
                const float f = m == -INFINITY ? 0.f : exp2_fast(m - M), inv = L == 0.f ? 0.f : 1.f / L;
                const int most = 16 / a.copies;        // columns that a thread adds up: 4 or 8
#pragma unroll 1
                for (int b = 0; b < HD / 16; ++b) {
                    uint32_t o[16];
                    ld16(o, to + 16 * b);
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) join[lane_row * 17 + i] = f == 0.f ? 0.f : __uint_as_float(o[i]) * f;
                    ok = group_sync(math_sync + x, syncs, gone);
                    if (!ok) break;
#pragma unroll 1
                    for (int i0 = copy * most; i0 < (copy + 1) * most; i0 += 4) {
                        float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                        for (int k = row; k < kRowTile; k += span)
#pragma unroll
                            for (int i = 0; i < 4; ++i) y[i] += join[k * 17 + i0 + i];
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] *= inv;
                        store4(16 * b + i0, y);
                    }
                    ok = group_sync(math_sync + x, syncs, gone);
                    if (!ok) break;
                }
                if (!ok) break;
                if (!whole && live && copy == 0)
                    a.part_lse[piece_at * a.unit_rows + ur] = L == 0.f ? -INFINITY : M + log2f(L);
            } else if (busy) {
                const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
                for (int b = 0; b < HD / 32; ++b) {
                    uint32_t o[32];
                    ld32(o, to + 32 * b);
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float y[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) y[k] = inv == 0.f ? 0.f : __uint_as_float(o[i + k]) * inv;
                        store4(32 * b + i, y);
                    }
                }
                if (!whole && live) a.part_lse[piece_at * a.unit_rows + ur] = l == 0.f ? -INFINITY : m + log2f(l);
            }
            g += n;
            ++seg;
        }
    }
    fence_before();
    __syncthreads();
    settle(gone);
    fence_after();
    if (warp == 12) tmem_free(tm, 512);
    if (threadIdx.x == 0 && *gone) atomicOr(a.err, kErrTcWait);
}

template <typename T, int HD, Rows ROWS>
int launch_rows(const Args& a, int blocks, cudaStream_t s) {
    if (!allow_smem<&k_cached_tc<T, HD, ROWS>>(Shape<HD>::SMEM)) return kErrCuda;
    k_cached_tc<T, HD, ROWS><<<blocks, kThreads, Shape<HD>::SMEM, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda;
}

template <typename T, int HD>
int launch(const Args& a, int blocks, cudaStream_t s) {
    const int st = a.copies > 1 ? launch_rows<T, HD, kCopies>(a, blocks, s)
                 : a.unit_rows <= kRowTile ? launch_rows<T, HD, kOneTile>(a, blocks, s)
                                           : launch_rows<T, HD, kTwoTiles>(a, blocks, s);
    return st ? st : launch_join<T, HD>(a, blocks, s);
}

template <typename T>
int by_dim(const Args& a, int blocks, cudaStream_t s) {
    switch (a.p.head_dim) {
        case 32: return launch<T, 32>(a, blocks, s);
        case 64: return launch<T, 64>(a, blocks, s);
        default: return launch<T, 128>(a, blocks, s);
    }
}

}  // namespace

size_t attention_cached_tc_workspace(int blocks, int nodes, int heads, int kv_heads, int head_dim) {
    return pieces_bytes(blocks, kUnitRows, nodes, heads, kv_heads, head_dim);
}

int attention_cached_tc(const CachedParams& p, int blocks, cudaStream_t s) {
    Args a{};
    if (int st = fill(a, p, kUnitRows, blocks)) return st;
    a.copies = a.unit_rows <= 32 ? 4 : a.unit_rows <= 64 ? 2 : 1;
    // What a unit's first scores and last sums take, measured: 64 decode calls 232 us
    // with 0, 219.5 with 1, 220 with 2; trees of two row tiles, which do not overlap
    // a unit's end with the next one's start, 148 with 0, 131, 123, 119.5 with 3, 120.5 with 4.
    a.start = a.unit_rows > kRowTile ? 3 : 1;
    return p.type == kBF16 ? by_dim<__nv_bfloat16>(a, blocks, s) : by_dim<__half>(a, blocks, s);
}

}  // namespace racb
