// cache_pages.cu -- the pages of a key/value cache: rows appended, pages
// copied, accepted rows of drafted trees moved together.
//
// Nothing is computed: each moved byte is read once and written once, in
// 16-byte units whatever the element type, and HBM bandwidth (launch latency
// for a few rows) bounds them.  96 pages of 256 KiB (k and v, 64 rows of 8 heads of
// 128, bf16) copied in each of 16 layers: 140 us, 5.8 TB/s read and written, 0.88
// of the copy peak.  4072 rows of them appended in one layer: 12 us; accepted
// rows of trees moved together: 10 us, the launch's time.  Page and row numbers come from device memory;
// one outside its range is skipped and sets the device error word.
#include "attn_common.cuh"

namespace racb {
namespace {

// Strides in 16-byte units.
struct Units { char* p; long long page, head, row, layer; };
Units units(const Pages& x, int type) {
    const int e = elem_bytes(type);
    return {static_cast<char*>(x.p), x.page * e, x.head * e, x.row * e, x.layer * e};
}
bool units_ok(const Pages& x, int type) {
    const int e = elem_bytes(type);
    return x.p && (reinterpret_cast<uintptr_t>(x.p) & 15u) == 0 && x.page * e % 16 == 0 && x.head * e % 16 == 0 &&
           x.row * e % 16 == 0 && x.layer * e % 16 == 0;
}

struct AppendArgs {
    Units k, v;
    const char *nk, *nv;
    long long nk_row, nk_head, nv_row, nv_head;
    const int *table, *starts, *cu;
    int table_width, pages, page_size, batch, kv_heads, vecs;
    long long tokens;
    unsigned int* err;
};

// One warp a new row: finds its sequence (a 32-way search in cu), then copies
// the row's heads of k and v.  Rows of 2 x 2 KiB keep 4072 warps' reads in flight.
__global__ void __launch_bounds__(256) k_cache_append(const AppendArgs a) {
    const long long tok = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (tok >= a.tokens) return;
    const int lo = warp_search(a.batch, tok, [&](int i) { return packed_cu(a.cu, i, a.tokens); });
    if (lo >= a.batch) return;                // behind the last sequence
    const long long row = (long long)a.starts[lo] + tok - packed_cu(a.cu, lo, a.tokens);
    const long long pi = row >= 0 ? row / a.page_size : -1;
    const int pg = pi >= 0 && pi < a.table_width ? a.table[(long long)lo * a.table_width + pi] : -1;
    if (pg < 0 || pg >= a.pages) {
        if (lane == 0) atomicOr(a.err, kErrBadPage);
        return;
    }
    const long long slot = row % a.page_size;
    const char *sk = a.nk + tok * a.nk_row, *sv = a.nv + tok * a.nv_row;
    char *dk = a.k.p + pg * a.k.page + slot * a.k.row, *dv = a.v.p + pg * a.v.page + slot * a.v.row;
    // Eight units a lane are read before the first is written: one trip to memory, not eight.
    const int n = 2 * a.kv_heads * a.vecs;
    for (int e0 = lane; e0 < n; e0 += 8 * 32) {
        uint4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = e0 + 32 * i, hk = e / a.vecs, c = e - hk * a.vecs, h = hk >> 1;
            if (e < n) x[i] = *reinterpret_cast<const uint4*>(hk & 1 ? sv + h * a.nv_head + c * 16 : sk + h * a.nk_head + c * 16);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = e0 + 32 * i, hk = e / a.vecs, c = e - hk * a.vecs, h = hk >> 1;
            if (e < n) *reinterpret_cast<uint4*>(hk & 1 ? dv + h * a.v.head + c * 16 : dk + h * a.k.head + c * 16) = x[i];
        }
    }
}

struct CopyArgs {
    Units x[2];
    const int *src, *dst;
    int pages, rows, heads, vecs;             // vecs 16-byte units a row
    unsigned int* err;
};

// Grid (parts of a page, page, layer and tensor).  A thread reads eight units
// before it writes the first.  FLAT: the page is one run of memory.
template <bool FLAT>
__global__ void __launch_bounds__(256) k_cache_copy(const CopyArgs a) {
    const Units& x = a.x[blockIdx.z & 1];
    const long long layer = blockIdx.z >> 1;
    const int from = a.src[blockIdx.y], to = a.dst[blockIdx.y];
    if (from < 0 || from >= a.pages || to < 0 || to >= a.pages) {
        if (threadIdx.x == 0) atomicOr(a.err, kErrBadPage);
        return;
    }
    const char* s = x.p + layer * x.layer + from * x.page;
    char* d = x.p + layer * x.layer + to * x.page;
    const int n = a.rows * a.heads * a.vecs;
    auto place = [&](int e) -> long long {
        if (FLAT) return (long long)e * 16;
        const int r = e / a.vecs, c = e - r * a.vecs, h = r / a.rows;
        return h * x.head + (r - h * a.rows) * x.row + c * 16;
    };
    const int e0 = blockIdx.x * 2048 + threadIdx.x;
    uint4 u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (e0 + 256 * i < n) u[i] = __ldcs(reinterpret_cast<const uint4*>(s + place(e0 + 256 * i)));
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (e0 + 256 * i < n) __stcs(reinterpret_cast<uint4*>(d + place(e0 + 256 * i)), u[i]);
}

struct CompactArgs {
    Units x[2];
    const int *table, *starts, *accepted, *n_accepted;
    int table_width, pages, page_size, nodes, vecs;
    unsigned int* err;
};

constexpr int kMaxNodes = 64, kMaxVecs = 32;  // 64 rows of 512 bytes: 32 KiB

// One CTA moves the rows of one (sequence, head) of one layer's k or v: all of
// them are read before the first is written, so the accepted nodes may come in
// any order.
__global__ void __launch_bounds__(256) k_cache_compact(const CompactArgs a) {
    __shared__ uint4 buf[kMaxNodes * kMaxVecs];
    __shared__ long long from[kMaxNodes], to[kMaxNodes];
    const int b = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
    const Units& x = a.x[blockIdx.z & 1];
    char* base = x.p + (long long)(blockIdx.z >> 1) * x.layer + head * x.head;
    const int n = max(0, min(a.n_accepted[b], a.nodes));
    if (tid < n) {
        const int acc = a.accepted[(long long)b * a.nodes + tid];
        long long at[2] = {-1, -1};
        bool bad = acc < 0 || acc >= a.nodes;
        if (!bad && acc != tid) {
            for (int i = 0; i < 2; ++i) {
                const long long row = (long long)a.starts[b] + (i ? tid : acc);
                const long long pi = row >= 0 ? row / a.page_size : -1;
                const int pg = pi >= 0 && pi < a.table_width ? a.table[(long long)b * a.table_width + pi] : -1;
                if (pg < 0 || pg >= a.pages) bad = true;
                else at[i] = pg * x.page + (row % a.page_size) * x.row;
            }
        }
        if (bad) { at[0] = at[1] = -1; atomicOr(a.err, kErrBadPage); }
        from[tid] = at[0];
        to[tid] = at[1];
    }
    __syncthreads();
    for (int e = tid; e < n * a.vecs; e += 256) {
        const int i = e / a.vecs, c = e % a.vecs;
        if (from[i] >= 0) buf[e] = *reinterpret_cast<const uint4*>(base + from[i] + c * 16);
    }
    __syncthreads();
    for (int e = tid; e < n * a.vecs; e += 256) {
        const int i = e / a.vecs, c = e % a.vecs;
        if (from[i] >= 0) *reinterpret_cast<uint4*>(base + to[i] + c * 16) = buf[e];
    }
}

int error_word(unsigned int** w) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return kErrCuda; }
    *w = device_error_word(dev);
    return *w ? kOk : kErrCuda;
}
int launched() { return cudaGetLastError() == cudaSuccess ? kOk : kErrCuda; }

bool shape_ok(int kv_heads, int head_dim, int pages, int page_size, int type) {
    return kv_heads > 0 && head_dim > 0 && pages >= 0 && page_size > 0 && type >= kF32 && type <= kBF16;
}

}  // namespace

int cache_append(const AppendParams& p, cudaStream_t s) {
    if (!shape_ok(p.kv_heads, p.head_dim, p.pages, p.page_size, p.type) || p.batch < 0 || p.tokens < 0 ||
        p.table_width < 0 || p.tokens >= (1LL << 31))
        return kErrInvalidDim;
    if (p.tokens == 0 || p.batch == 0) return kOk;
    const int e = elem_bytes(p.type);
    if (!p.k.p || !p.v.p || !p.nk.p || !p.nv.p || !p.table || !p.starts || !p.cu) return kErrNullPtr;
    if (!units_ok(p.k, p.type) || !units_ok(p.v, p.type) || p.head_dim * e % 16) return kErrUnsupported;
    for (const Rows* r : {&p.nk, &p.nv})
        if ((reinterpret_cast<uintptr_t>(r->p) & 15u) || r->row * e % 16 || r->head * e % 16) return kErrUnsupported;
    AppendArgs a{units(p.k, p.type), units(p.v, p.type), static_cast<const char*>(p.nk.p),
                 static_cast<const char*>(p.nv.p), p.nk.row * e, p.nk.head * e, p.nv.row * e, p.nv.head * e,
                 p.table, p.starts, p.cu, p.table_width, p.pages, p.page_size, p.batch, p.kv_heads,
                 p.head_dim * e / 16, p.tokens, nullptr};
    if (int st = error_word(&a.err)) return st;
    k_cache_append<<<(unsigned)((p.tokens + 7) / 8), 256, 0, s>>>(a);
    return launched();
}

int cache_copy_pages(const CopyPagesParams& p, cudaStream_t s) {
    if (!shape_ok(p.kv_heads, p.head_dim, p.pages, p.page_size, p.type) || p.n < 0 || p.layers < 0 || p.n > 65535 ||
        p.layers > 32767)
        return kErrInvalidDim;
    if (p.n == 0 || p.layers == 0) return kOk;
    const int e = elem_bytes(p.type);
    if (!p.k.p || !p.v.p || !p.src || !p.dst) return kErrNullPtr;
    if (!units_ok(p.k, p.type) || !units_ok(p.v, p.type) || p.head_dim * e % 16) return kErrUnsupported;
    CopyArgs a{{units(p.k, p.type), units(p.v, p.type)}, p.src, p.dst, p.pages, p.page_size, p.kv_heads,
               p.head_dim * e / 16, nullptr};
    if (int st = error_word(&a.err)) return st;
    const long long vecs = (long long)a.rows * a.heads * a.vecs;
    if (vecs >= (1LL << 31)) return kErrInvalidDim;
    const unsigned parts = (unsigned)((vecs + 2047) / 2048);
    const dim3 grid(parts, p.n, 2 * p.layers);
    const auto flat = [&](const Pages& x) { return x.row == p.head_dim && x.head == (long long)p.page_size * x.row; };
    if (flat(p.k) && flat(p.v)) k_cache_copy<true><<<grid, 256, 0, s>>>(a);
    else k_cache_copy<false><<<grid, 256, 0, s>>>(a);
    return launched();
}

int cache_compact(const CompactParams& p, cudaStream_t s) {
    if (!shape_ok(p.kv_heads, p.head_dim, p.pages, p.page_size, p.type) || p.batch < 0 || p.nodes < 0 ||
        p.nodes > kMaxNodes || p.layers < 0 || p.layers > 32767 || p.table_width < 0 || p.kv_heads > 65535)
        return kErrInvalidDim;
    if (p.batch == 0 || p.nodes == 0 || p.layers == 0) return kOk;
    const int e = elem_bytes(p.type);
    if (!p.k.p || !p.v.p || !p.table || !p.starts || !p.accepted || !p.n_accepted) return kErrNullPtr;
    if (!units_ok(p.k, p.type) || !units_ok(p.v, p.type) || p.head_dim * e % 16 || p.head_dim * e / 16 > kMaxVecs)
        return kErrUnsupported;
    CompactArgs a{{units(p.k, p.type), units(p.v, p.type)}, p.table, p.starts, p.accepted, p.n_accepted,
                  p.table_width, p.pages, p.page_size, p.nodes, p.head_dim * e / 16, nullptr};
    if (int st = error_word(&a.err)) return st;
    k_cache_compact<<<dim3(p.batch, p.kv_heads, 2 * p.layers), 256, 0, s>>>(a);
    return launched();
}

}  // namespace racb
