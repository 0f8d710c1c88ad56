// attention_packed.cu -- attention over packed prompts, forward and backward:
// arguments, workspace, and the choice of kernels by type.
//
// Sequences of different lengths lie end to end in [tokens, heads, head_dim];
// query head h reads key/value head h / (heads / kv_heads).  Within a sequence
//   s_ij = scale q_i . k_j,  j <= i when causal,  p_ij = exp(s_ij - lse_i),
//   lse_i = log sum_j exp(s_ij),  o_i = sum_j p_ij v_j,
// and with do the output's gradient, D_i = do_i . o_i, ds_ij = p_ij (do_i . v_j - D_i):
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_{h,i} ds_ij q_i,  dv_j = sum_{h,i} p_ij do_i
// (sums over the query heads h that share the key/value head).  Every sum is
// held in 32 bits, in a fixed order: no atomics on sums, the same bits every time.
#include "attn_common.cuh"

namespace racb {
namespace {

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
        packed_slots(p.tokens, p.n_seqs, 128) * (2 * p.heads + 2 * p.kv_heads) >= (1LL << 31))
        return kErrInvalidDim;
    if (p.tokens && (!p.q.p || !p.k.p || !p.v.p || (p.n_seqs && !p.cu))) return kErrNullPtr;
    if (!rows_ok(p.q, p.type) || !rows_ok(p.k, p.type) || !rows_ok(p.v, p.type)) return kErrUnsupported;
    return kOk;
}

}  // namespace

// 16-bit types, backward: D, [heads, tokens], and two largest values of each sequence and key/value head.
size_t attention_packed_workspace(long long tokens, int n_seqs, int heads, int kv_heads, int head_dim, int type,
                                  int backward) {
    if (type == kF32) return attention_packed_f32_workspace(tokens, n_seqs, heads, kv_heads, head_dim, backward);
    return backward ? sizeof(float) * ((size_t)tokens * heads + 2 * (size_t)n_seqs * kv_heads) : 0;
}

static bool room_ok(const PackedParams& p, int backward) {
    const size_t n = attention_packed_workspace(p.tokens, p.n_seqs, p.heads, p.kv_heads, p.head_dim, p.type, backward);
    return n == 0 || (p.ws && p.ws_bytes >= n && (reinterpret_cast<uintptr_t>(p.ws) & 15u) == 0);
}

// A thread of autograd's may have no context yet, which the tensor maps need.
static int bind_device() {
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) return kOk;
    cudaGetLastError();
    return kErrCuda;
}

int attention_packed(const PackedParams& p, cudaStream_t s) {
    if (int st = check(p)) return st;
    if (p.tokens == 0) return kOk;
    if (!p.out) return kErrNullPtr;
    if ((reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.low)) & 15u) return kErrUnsupported;
    if (!room_ok(p, 0)) return kErrAlloc;
    if (int st = bind_device()) return st;
    return p.type == kF32 ? attention_packed_f32(p, 0, s) : attention_packed_tc(p, s);
}

int attention_packed_backward(const PackedParams& p, cudaStream_t s) {
    if (int st = check(p)) return st;
    if (p.tokens == 0) return kOk;
    if (!p.dout.p || !p.out_in || !p.lse_in || !p.dq || !p.dk || !p.dv) return kErrNullPtr;
    if (!rows_ok(p.dout, p.type)) return kErrUnsupported;
    if (!room_ok(p, 1)) return kErrAlloc;
    for (const void* x : {p.out_in, (const void*)p.low, (const void*)p.dq, (const void*)p.dk, (const void*)p.dv})
        if (reinterpret_cast<uintptr_t>(x) & 15u) return kErrUnsupported;
    if (int st = bind_device()) return st;
    return p.type == kF32 ? attention_packed_f32(p, 1, s) : attention_packed_backward_tc(p, s);
}

}  // namespace racb
