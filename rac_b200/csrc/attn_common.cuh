// attn_common.cuh -- what the packed-prompt and the paged-cache attention
// kernels share: element types, the tile map of packed sequences, the row map
// of paged caches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "attn_ops.h"
#include "rac_internal.h"

namespace racb {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Four consecutive elements as floats (16- or 8-byte aligned source).
__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <typename T> __device__ __forceinline__ float4 load4(const T* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
    return make_float4(to_f32(e[0]), to_f32(e[1]), to_f32(e[2]), to_f32(e[3]));
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
template <typename T> __device__ __forceinline__ void store4(T* p, float4 v) {
    T e[4] = {from_f32<T>(v.x), from_f32<T>(v.y), from_f32<T>(v.z), from_f32<T>(v.w)};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(e);
}

// Raises a kernel's limit of dynamic shared memory, once for each device.
template <auto* Kernel>
bool allow_smem(int bytes) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return false; }
    if (done.load(std::memory_order_relaxed) >> dev & 1) return true;
    if (cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return true;
}

// ── packed sequences ──────────────────────────────────────────────────────
// Sequence i holds rows [cu[i], cu[i+1]) of the packed tensors.  Tiles of BM
// rows never cross a sequence, and the host does not know the lengths (reading
// them would stall the stream), so the grid has a slot for every tile that any
// lengths could need: sequence i owns the slots from cu[i] / BM + i on, because
// floor(a / BM) + ceil(b / BM) <= floor((a + b) / BM) + 1.  tokens / BM + n + 1
// slots cover every sequence and, after the last one, the rows behind it
// (seq == n).  cu is read clamped to [0, tokens] with cu[0] taken as 0, so no
// contents of cu lead outside the tensors.
struct PackedTile {
    int seq;             // n: rows behind the last sequence
    long long start;     // first row of the sequence
    int len;             // its rows
    int row0;            // first row of the tile within the sequence (>= len: no tile)
};

__host__ __device__ inline long long packed_slots(long long tokens, int n, int bm) { return tokens / bm + n + 1; }

__device__ __forceinline__ long long packed_cu(const int* __restrict__ cu, int i, long long tokens) {
    if (i == 0) return 0;
    const long long v = __ldg(cu + i);
    return v < 0 ? 0 : (v > tokens ? tokens : v);
}

// The largest i in [0, n] with key(i) <= x, key rising and key(0) <= x.  Called
// by whole warps: a 32-way search, one step up to 31 sequences.
template <typename F>
__device__ __forceinline__ int warp_search(int n, long long x, F key) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n;
    while (hi > lo) {
        const int step = (hi - lo + 31) / 32;
        const long long i = lo + (long long)(lane + 1) * step;
        const bool le = i <= hi && key((int)(i <= hi ? i : hi)) <= x;
        lo += __popc(__ballot_sync(0xffffffffu, le)) * step;
        hi = min(hi, lo + step - 1);
    }
    return lo;
}

__device__ __forceinline__ PackedTile packed_tile(const int* __restrict__ cu, int n, long long tokens, int bm,
                                                  long long slot) {
    const int lo = warp_search(n, slot, [&](int i) { return packed_cu(cu, i, tokens) / bm + i; });
    PackedTile t;
    t.seq = lo;
    t.start = packed_cu(cu, lo, tokens);
    const long long end = lo < n ? packed_cu(cu, lo + 1, tokens) : tokens;
    t.len = (int)(end > t.start ? end - t.start : 0);
    const long long r = (slot - (t.start / bm + lo)) * bm;
    t.row0 = (int)(r < 0 || r > t.len ? t.len : r);
    return t;
}

// ── paged caches ──────────────────────────────────────────────────────────
// Row r of sequence b lies in page table[b][r / page], slot r % page.  A page
// number outside [0, pages) is never followed: the row counts as hidden and
// the device error word is set (RAC_ERR_DEVICE at the next check).
constexpr unsigned int kErrBadPage = 8u;   // bit 3 of the device error word

}  // namespace racb
