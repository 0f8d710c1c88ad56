"""Torch-tensor front end of librac_b200.so.

The first half mirrors the pybind surface of the reference extension
``rac_cuda_ext`` (rac_torch/rac_torch_bind.cpp:223-258 and
rac_torch/rac_torch.cu:1181-1214): same function names, argument names,
defaults and conventions --

* ``iters <= 0`` takes the process-wide iteration knob, ``mode < 0`` the
  process-wide mode (rac_torch_bind.cpp:81-82);
* fp16/bf16 inputs are computed in fp32 and cast back (rac_torch.cu:867-872);
* an empty bias tensor means "no bias";
* kernels run on the current torch CUDA stream.

The second half exposes the elementwise / row-wise kernels on tensors.
Every call needs CUDA tensors: there is no CPU path, and a CPU tensor is a
``ValueError``.
"""
from __future__ import annotations

import contextlib
import functools

import torch

from . import _lib
from ._lib import LAYOUT_NN, LAYOUT_NT, LAYOUT_TN

MODE_FAST, MODE_CORDIC, MODE_SHIFTADD = 0, 1, 2
ACT_NONE, ACT_RELU, ACT_GELU, ACT_SILU = 0, 1, 2, 3
# silu(v[:, 2c]) * v[:, 2c+1] over row-interleaved gate/up weights (N/2 outputs)
ACT_SWIGLU = 4

# Process-wide knobs of the torch binding (rac_torch_bind.cpp:54-55):
# defaults iters = 24, mode = FAST.
_iters = 24
_mode = MODE_FAST


def set_cordic_iters(iters: int) -> None:
    """rac_torch_bind.cpp:205-212: <= 0 resets to 24, else clamp to [1, 24]."""
    global _iters
    _iters = 24 if iters <= 0 else max(1, min(24, int(iters)))


def get_cordic_iters() -> int:
    return _iters


def set_cordic_mode(mode: int) -> None:
    """rac_torch_bind.cpp:216-219: unknown modes fall back to FAST."""
    global _mode
    _mode = mode if mode in (MODE_FAST, MODE_CORDIC, MODE_SHIFTADD) else MODE_FAST


def get_cordic_mode() -> int:
    return _mode


def _resolve(iters: int, mode: int) -> tuple[int, int]:
    it = _iters if iters <= 0 else max(1, min(24, int(iters)))
    md = _mode if mode < 0 else int(mode)
    return it, md


def _need_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("librac_b200 runs on CUDA tensors only (no CPU path)")


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _f32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float32 else t.float()


def _ptr(t):
    return None if t is None else t.data_ptr()


def gemm(A: torch.Tensor, B: torch.Tensor, layout: int = LAYOUT_NN, iters: int = 0,
         mode: int = -1, bias: torch.Tensor | None = None, act: int = ACT_NONE,
         residual: torch.Tensor | None = None, alpha: float = 1.0, beta: float | None = None,
         out: torch.Tensor | None = None, variant: int = 0) -> torch.Tensor:
    """C = act(alpha * op(A) op(B) + beta * residual + bias) for 2-D fp32 CUDA tensors.

    layout NN: A[M,K] B[K,N]; NT: A[M,K] B[N,K]; TN: A[K,M] B[K,N].
    Inner (last) dims must be contiguous; leading dims may be strided."""
    _need_cuda(A, B, bias, residual)
    it, md = _resolve(iters, mode)
    A, B = _f32(A), _f32(B)
    if A.dim() != 2 or B.dim() != 2:
        raise ValueError("gemm: 2-D operands required")
    if A.stride(1) != 1:
        A = A.contiguous()
    if B.stride(1) != 1:
        B = B.contiguous()
    if layout == LAYOUT_TN:
        K, M = A.shape
    else:
        M, K = A.shape
    N = B.shape[0] if layout == LAYOUT_NT else B.shape[1]
    Kb = B.shape[1] if layout == LAYOUT_NT else B.shape[0]
    if Kb != K:
        raise ValueError(f"gemm: inner dimensions differ ({K} vs {Kb})")
    if act == ACT_SWIGLU:
        if N % 2 or residual is not None or (beta or 0.0) != 0.0:
            raise ValueError("gemm: SwiGLU needs an even N and no residual")
    if out is None:
        out = torch.empty((M, N // 2 if act == ACT_SWIGLU else N), device=A.device,
                          dtype=torch.float32)
    if residual is not None:
        residual = _f32(residual)
        if residual.stride(-1) != 1:
            residual = residual.contiguous()
        b = 1.0 if beta is None else float(beta)
    else:
        b = 0.0 if beta is None else float(beta)
        if b != 0.0:
            residual = out
    if bias is not None:
        bias = _f32(bias).contiguous()
        if bias.numel() == 0:
            bias = None
    if M == 0 or N == 0:
        return out
    if K == 0:
        return out.zero_() if residual is None else out.copy_(residual).mul_(b)
    with torch.cuda.device(A.device):
        _lib.call("rac_gemm_async", _ptr(A), A.stride(0), _ptr(B), B.stride(0), _ptr(out),
                  out.stride(0), _ptr(residual), residual.stride(0) if residual is not None else 0,
                  _ptr(bias), M, N, K, layout, md, it, float(alpha), b, act, variant, _stream(A))
    return out


# ── rac_cuda_ext surface ───────────────────────────────────────────────────

def matmul_forward(A: torch.Tensor, B: torch.Tensor, iters: int = 0, mode: int = -1) -> torch.Tensor:
    """rac_torch_bind.cpp:61-88: C = A @ B (NN)."""
    if A.dim() != 2 or B.dim() != 2 or A.shape[1] != B.shape[0]:
        raise ValueError("RAC: 2D tensors with matching inner dimension required")
    dt = A.dtype
    C = gemm(A.contiguous(), B.contiguous(), LAYOUT_NN, iters, mode)
    return C if dt == torch.float32 else C.to(dt)


def matmul_backward(grad_C, A, B, need_grad_A=True, need_grad_B=True, iters=0, mode=-1):
    """rac_torch_bind.cpp:130-162: dA = dC @ B^T (NT), dB = A^T @ dC (TN)."""
    gC, A_, B_ = _f32(grad_C).contiguous(), _f32(A).contiguous(), _f32(B).contiguous()
    gA = gemm(gC, B_, LAYOUT_NT, iters, mode) if need_grad_A else None
    gB = gemm(A_, gC, LAYOUT_TN, iters, mode) if need_grad_B else None
    if gA is not None and A.dtype != torch.float32:
        gA = gA.to(A.dtype)
    if gB is not None and B.dtype != torch.float32:
        gB = gB.to(B.dtype)
    return [gA, gB]


def linear_forward(input, weight, bias, iters=0, mode=-1, act: int = ACT_NONE,
                   residual: torch.Tensor | None = None):
    """rac_torch_bind.cpp:90-128: out = input @ weight^T + bias (NT), bias and an
    optional activation / residual add fused into the GEMM epilogue."""
    dt = input.dtype
    shape = list(input.shape)
    x2 = input.reshape(-1, weight.shape[1])
    r2 = residual.reshape(-1, weight.shape[0]) if residual is not None else None
    out = gemm(x2, weight, LAYOUT_NT, iters, mode,
               bias=bias if (bias is not None and bias.numel() > 0) else None,
               act=act, residual=r2)
    shape[-1] = weight.shape[0] // 2 if act == ACT_SWIGLU else weight.shape[0]
    out = out.reshape(shape)
    return out if dt == torch.float32 else out.to(dt)


def linear_backward(grad_output, input, weight, need_bias_grad, iters=0, mode=-1):
    """rac_torch_bind.cpp:164-199: grad_input (NN), grad_weight (TN), grad_bias."""
    out_f, in_f = weight.shape
    go = _f32(grad_output).reshape(-1, out_f).contiguous()
    inp = _f32(input).reshape(-1, in_f).contiguous()
    gi = gemm(go, _f32(weight).contiguous(), LAYOUT_NN, iters, mode)
    gw = gemm(go, inp, LAYOUT_TN, iters, mode)
    gb = go.sum(0) if need_bias_grad else None
    return [gi.reshape(list(input.shape[:-1]) + [in_f]), gw, gb]


def fused_linear_forward(input, weight, bias, act, iters=0, mode=-1):
    """rac_torch.cu:1037-1086: act(input @ weight^T + bias) in one kernel."""
    return linear_forward(input, weight, bias, iters, mode, act=int(act))


def act_grad(pre_act: torch.Tensor, act: int) -> torch.Tensor:
    """Derivative of the activation at pre_act (rac_torch.cu:680-697)."""
    x = pre_act.float()
    if act == ACT_RELU:
        return (x > 0).float()
    if act == ACT_GELU:
        cdf = 0.5 * (1.0 + torch.erf(x * 0.7071067811865))
        pdf = 0.3989422804 * torch.exp(-0.5 * x * x)
        return cdf + x * pdf
    if act == ACT_SILU:
        sig = torch.sigmoid(x)
        return sig * (1.0 + x * (1.0 - sig))
    return torch.ones_like(x)


def fused_linear_backward(grad_output, input, weight, bias, pre_act, act, has_bias,
                          iters=0, mode=-1):
    """rac_torch.cu:1093-1177: gradient through act, then the linear backward."""
    d = _f32(grad_output) * act_grad(pre_act, int(act))
    gi, gw, gb = linear_backward(d, input, weight, bool(has_bias), iters, mode)
    return [gi, gw, gb]


# ── elementwise and row-wise kernels on tensors ───────────────────────────

def _prep(t: torch.Tensor) -> torch.Tensor:
    _need_cuda(t)
    if t.dtype != torch.float32:
        raise ValueError("float32 tensor required")
    return t.contiguous()


def rotate_batch(v: torch.Tensor, theta: torch.Tensor, iters: int | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """v[..., 2] rotated by theta[...]: rac_rotate_batch (iters None: literal
    RAC_K_INV, 16 iterations, lib/c/rac_cpu.c:136-139) or rac_rotate_n."""
    v, theta = _prep(v), _prep(theta)
    if v.shape[-1] != 2 or v.numel() != 2 * theta.numel():
        raise ValueError("v must be [..., 2] with one angle per vector")
    out = torch.empty_like(v) if out is None else out
    lit = 1 if iters is None else 0
    with torch.cuda.device(v.device):
        _lib.call("rac_rotate_batch_async", v.data_ptr(), theta.data_ptr(), out.data_ptr(),
                  theta.numel(), 16 if iters is None else int(iters), lit, _stream(v))
    return out


def project_batch(v: torch.Tensor, theta: torch.Tensor, iters: int = 16) -> torch.Tensor:
    """rac_project_n per element (lib/c/rac_cpu.c:282-288)."""
    v, theta = _prep(v), _prep(theta)
    if v.shape[-1] != 2 or v.numel() != 2 * theta.numel():
        raise ValueError("v must be [..., 2] with one angle per vector")
    out = torch.empty_like(theta)
    with torch.cuda.device(v.device):
        _lib.call("rac_project_batch_async", v.data_ptr(), theta.data_ptr(), out.data_ptr(),
                  theta.numel(), int(iters), _stream(v))
    return out


def sincos(theta: torch.Tensor):
    """rac_sincos per element: (sin, cos)."""
    theta = _prep(theta)
    s, c = torch.empty_like(theta), torch.empty_like(theta)
    with torch.cuda.device(theta.device):
        _lib.call("rac_sincos_batch_async", theta.data_ptr(), s.data_ptr(), c.data_ptr(),
                  theta.numel(), _stream(theta))
    return s, c


def _unary(x: torch.Tensor, op: int) -> torch.Tensor:
    x = _prep(x)
    y = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.call("rac_unary_async", x.data_ptr(), y.data_ptr(), x.numel(), op, _stream(x))
    return y


def exp(x):
    return _unary(x, _lib.UNARY_EXP)


def tanh(x):
    return _unary(x, _lib.UNARY_TANH)


def rsqrt(x):
    return _unary(x, _lib.UNARY_RSQRT)


def sigmoid(x):
    return _unary(x, _lib.UNARY_SIGMOID)


def softmax(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Row softmax over the last dim (lib/c/rac_cpu.c:258-271)."""
    x = _prep(x)
    y = torch.empty_like(x) if out is None else out
    d = x.shape[-1]
    with torch.cuda.device(x.device):
        _lib.call("rac_softmax_async", x.data_ptr(), y.data_ptr(), x.numel() // max(d, 1), d,
                  _stream(x))
    return y


def rmsnorm(x: torch.Tensor, gamma: torch.Tensor | None = None, eps: float = 1e-6,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """lib/c/rac_cpu.c:548-574 over the last dim."""
    x = _prep(x)
    g = _prep(gamma) if gamma is not None else None
    y = torch.empty_like(x) if out is None else out
    d = x.shape[-1]
    with torch.cuda.device(x.device):
        _lib.call("rac_rmsnorm_async", x.data_ptr(), y.data_ptr(), _ptr(g), float(eps),
                  x.numel() // max(d, 1), d, _stream(x))
    return y


def layernorm(x, gamma=None, beta=None, eps: float = 1e-5,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """lib/c/rac_cpu.c:507-546 over the last dim."""
    x = _prep(x)
    g = _prep(gamma) if gamma is not None else None
    b = _prep(beta) if beta is not None else None
    y = torch.empty_like(x) if out is None else out
    d = x.shape[-1]
    with torch.cuda.device(x.device):
        _lib.call("rac_layernorm_async", x.data_ptr(), y.data_ptr(), _ptr(g), _ptr(b), float(eps),
                  x.numel() // max(d, 1), d, _stream(x))
    return y


def rope_cache(max_seq: int, head_dim: int, base: float = 10000.0, device="cuda"):
    """rac_rope_cache (lib/c/rac_cpu.c:576-598): (cos, sin) [max_seq, head_dim/2]."""
    c = torch.empty((max_seq, head_dim // 2), device=device, dtype=torch.float32)
    s = torch.empty_like(c)
    with torch.cuda.device(c.device):
        _lib.call("rac_rope_cache_async", c.data_ptr(), s.data_ptr(), max_seq, head_dim,
                  float(base), _stream(c))
    return c, s


def rope_apply_(x: torch.Tensor, cos_tab: torch.Tensor, sin_tab: torch.Tensor,
                positions: torch.Tensor | None = None, form: int = 0) -> torch.Tensor:
    """In place on contiguous x[..., seq, head_dim]. form 0 = lib/c fmaf form,
    1 = torch RACRoPE form.  positions: optional int index per seq row."""
    _need_cuda(x)
    if not x.is_contiguous() or x.dtype != torch.float32:
        raise ValueError("rope_apply_ needs a contiguous float32 tensor")
    seq, hd = x.shape[-2], x.shape[-1]
    ct, st = _prep(cos_tab), _prep(sin_tab)
    pos = positions.to(device=x.device, dtype=torch.int32).contiguous() if positions is not None else None
    with torch.cuda.device(x.device):
        _lib.call("rac_rope_apply_async", x.data_ptr(), ct.data_ptr(), st.data_ptr(), _ptr(pos),
                  x.numel() // (seq * hd), seq, hd, int(form), _stream(x))
    return x


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: torch.Tensor | None = None,
              is_causal: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Fused softmax(q k^T / sqrt(hd) + mask) v on [B, H, S, hd] (rac_attention)."""
    q, k, v = _prep(q), _prep(k), _prep(v)
    m = _prep(mask) if mask is not None else None
    if m is not None and m.shape != (q.shape[-2], q.shape[-2]):
        raise ValueError("attention mask must be [seq, seq]")
    o = torch.empty_like(q) if out is None else out
    b, h, s_, hd = q.shape
    with torch.cuda.device(q.device):
        _lib.call("rac_attention_async", q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(m),
                  int(bool(is_causal)), o.data_ptr(), b, h, s_, hd, _stream(q))
    return o


# ── packed prompts and paged caches ───────────────────────────────────────

_ELEM = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_NEW_ROWS = 64            # new rows of a sequence that attention_cached takes (bits of a tree mask)
_DIMS = (32, 64, 128)
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") \
    else lambda i: torch.cuda.current_stream(i).cuda_stream


def _launch(name: str, args: bytes, device: int) -> None:
    """Calls an entry point that takes an argument structure, on the device's current stream."""
    if torch.cuda.current_device() == device:
        _lib.call(name, args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            _lib.call(name, args, _raw_stream(device))


def _elem(t: torch.Tensor, *more: torch.Tensor) -> int:
    dt = t.dtype
    e = _ELEM.get(dt)
    if e is None:
        raise ValueError(f"float32, float16 or bfloat16 tensors required, got {dt}")
    for x in more:
        if x.dtype is not dt:
            raise ValueError(f"tensors of one type required, got {t.dtype} and {x.dtype}")
    return e


def _device(t: torch.Tensor, *more: torch.Tensor | None) -> int:
    d = t.get_device()
    if d < 0:
        _need_cuda(t)
    for x in more:
        if x is not None and x.get_device() != d:
            _need_cuda(x)
            raise ValueError("tensors on one device required")
    return d


def _fits(t: torch.Tensor) -> bool:
    """Whether the kernels take t as it lies: contiguous last axis, 16-byte aligned base and strides, no axis
    expanded."""
    e = t.element_size()
    return (t.shape[-1] == 1 or t.stride(-1) == 1) and t.data_ptr() % 16 == 0 and all(
        s > 0 and s * e % 16 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)


def _rows(t: torch.Tensor, width: int) -> tuple:
    """(t or an aligned copy, its address, strides of its outer axes) for elements of `width` bytes; t has three
    or four axes."""
    x = t.data_ptr()
    s = t.stride()
    if len(s) == 3:
        a, b, c = s
        if not (x | a * width | b * width) & 15 and c == 1 and a and b:
            return t, x, (a, b)
    else:
        a, b, c, e = s
        if not (x | a * width | b * width | c * width) & 15 and e == 1 and a and b and c:
            return t, x, (a, b, c)
    if not _fits(t):
        t = t.clone(memory_format=torch.contiguous_format)
    # The stride of an axis of one place may be anything.
    return t, t.data_ptr(), tuple(v if n > 1 else 0 for v, n in zip(t.stride()[:-1], t.shape))


def _index(name: str, t: torch.Tensor, shape: tuple, dtype=torch.int32) -> torch.Tensor:
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype is not dtype:
        if t.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} must hold int32 or int64, got {t.dtype}")
        t = t.to(dtype)
    return t if t.is_contiguous() else t.contiguous()


def _check_heads(heads: int, kv_heads: int, hd: int) -> None:
    if hd not in _DIMS:
        raise ValueError(f"head size 32, 64 or 128 required, got {hd}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"the query heads ({heads}) must be a multiple of the key/value heads ({kv_heads})")


def _page_strides(t: torch.Tensor, width: int) -> tuple:
    """Strides of the outer axes of a page tensor, which the kernels take as it lies."""
    s = t.stride()
    y = t.data_ptr()
    for v in s[:-1]:
        y |= v * width
    if (y & 15 or s[-1] != 1 or 0 in s) and not _fits(t):
        raise ValueError("pages need a contiguous last axis and 16-byte aligned rows")
    return s[:-1]


def _check_out(name: str, out: torch.Tensor, shape: tuple, dtype) -> None:
    if out.shape != shape or out.dtype is not dtype or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"{name} must be a contiguous, 16-byte aligned {tuple(shape)} of {dtype}")


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def _check_packed(q, k, v, cu_seqlens):
    """(element type, cu_seqlens as int32, tokens, heads, kv_heads, dim)"""
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3:
        raise ValueError("attention_packed: q [tokens, heads, dim] and k, v [tokens, kv_heads, dim] required")
    t, h, hd = qs
    if v.shape != ks or ks[0] != t or ks[2] != hd:
        raise ValueError(f"attention_packed: shapes {tuple(qs)}, {tuple(ks)}, {tuple(v.shape)} differ")
    _check_heads(h, ks[1], hd)
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("attention_packed: cu_seqlens must be 1-D and start with 0")
    return _elem(q, k, v), _index("cu_seqlens", cu_seqlens, cu_seqlens.shape), t, h, ks[1], hd


def _packed_workspace(like, device, *sizes):
    n = 0
    if sizes[-2] == 0 or sizes[-1]:
        # Its size goes by the device's SMs.
        with contextlib.nullcontext() if torch.cuda.current_device() == device else torch.cuda.device(device):
            n = _lib.lib().rac_attention_packed_workspace(*sizes)
    return (like.new_empty(n, dtype=torch.uint8), n) if n else (None, 0)


def attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     is_causal: bool = True, scale: float | None = None, out: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None, out_low: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v within each sequence of a packed batch, on q [tokens, heads, dim] and
    k, v [tokens, kv_heads, dim] (float32, float16 or bfloat16; dim 32, 64 or 128; head h reads key/value
    head h // (heads // kv_heads)).  Sequence i holds rows cu_seqlens[i] .. cu_seqlens[i + 1] - 1; cu_seqlens
    starts with 0 and rises, lengths of 0 are allowed.  It stays on the device: its values are not checked,
    and no values lead outside the tensors.  scale None is dim ** -0.5.

    Rows behind the last sequence keep what `out` holds; without `out` they are zeros.  What lies in another
    sequence, NaN included, reaches no row.  (Within a sequence a NaN or an infinity in v reaches every row of
    the 128 whose keys it stands among, hidden or not.)
    float32: values are taken to 22 bits or, where that is more, 2^-39 of the largest finite one among 128 rows of
    a sequence's head, hidden ones included.

    For attention_packed_backward: `lse`, a float32 [heads, tokens], receives the logarithm of each row's sum.
    `out_low`, like out and of use in 16 bits, receives what rounding took from the first 128 rows of each
    sequence, where few keys share the weight: with it the gradients are rounded about as much as the output,
    without it short sequences' are up to twice as far off."""
    elem, cu, t, h, kv, hd = _check_packed(q, k, v, cu_seqlens)
    if out is not None:
        _check_out("out", out, q.shape, q.dtype)
    if lse is not None:
        _check_out("lse", lse, (h, t), torch.float32)
    if out_low is not None:
        _check_out("out_low", out_low, q.shape, q.dtype)
    d = _device(q, k, v, cu, out, lse, out_low)
    w = 2 if elem else 4
    q, qp, qs = _rows(q, w)
    k, kp, ks = _rows(k, w)
    v, vp, vs = _rows(v, w)
    o = _like(q) if out is None else out
    n = cu.shape[0] - 1
    ws, ws_n = _packed_workspace(q, d, t, n, h, kv, hd, elem, 0)
    _launch("rac_attention_packed_async", _lib.PACKED_ARGS.pack(
        qp, kp, vp, cu.data_ptr(), o.data_ptr(), 0 if lse is None else lse.data_ptr(),
        0 if out_low is None else out_low.data_ptr(), 0, 0, 0, 0,
        ws.data_ptr() if ws_n else 0, *qs, *ks, *vs, 0, 0, t, ws_n, n, h, kv, hd, elem, bool(is_causal), out is None,
        hd ** -0.5 if scale is None else scale), d)
    return o


def attention_packed_backward(grad_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                              out: torch.Tensor, lse: torch.Tensor, cu_seqlens: torch.Tensor,
                              is_causal: bool = True, scale: float | None = None,
                              out_low: torch.Tensor | None = None):
    """Gradients (dq, dk, dv) of attention_packed from its out, lse and out_low; the key/value heads' sum over the
    query heads that read them.  Rows behind the last sequence get zeros.  The same inputs give the same bits."""
    elem, cu, t, h, kv, hd = _check_packed(q, k, v, cu_seqlens)
    if grad_out.shape != q.shape:
        raise ValueError(f"grad_out must be {tuple(q.shape)}, got {tuple(grad_out.shape)}")
    _elem(q, grad_out)
    _check_out("out", out, q.shape, q.dtype)
    _check_out("lse", lse, (h, t), torch.float32)
    if out_low is not None:
        _check_out("out_low", out_low, q.shape, q.dtype)
    d = _device(q, k, v, cu, grad_out, out, lse, out_low)
    w = 2 if elem else 4
    q, qp, qs = _rows(q, w)
    k, kp, ks = _rows(k, w)
    v, vp, vs = _rows(v, w)
    g, gp, gs = _rows(grad_out, w)
    dq, dk, dv = _like(q), _like(k), _like(v)
    n = cu.shape[0] - 1
    ws, ws_n = _packed_workspace(q, d, t, n, h, kv, hd, elem, 1)
    _launch("rac_attention_packed_backward_async", _lib.PACKED_ARGS.pack(
        qp, kp, vp, cu.data_ptr(), out.data_ptr(), lse.data_ptr(), 0 if out_low is None else out_low.data_ptr(), gp, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
        ws.data_ptr() if ws_n else 0, *qs, *ks, *vs, *gs, t, ws_n, n, h, kv, hd, elem, bool(is_causal), 1,
        hd ** -0.5 if scale is None else scale), d)
    return dq, dk, dv


def _check_pages(k_pages, v_pages, elem: int, layers: bool):
    """(strides [layer,] page, head, row of k, of v, pages, kv_heads, page_size, dim) of two page tensors."""
    s = k_pages.shape
    n = len(s)
    if n != 4 and not (layers and n == 5) or v_pages.shape != s:
        raise ValueError("k_pages and v_pages must be alike, " + ("[[layers,] " if layers else "[") +
                         "pages, kv_heads, page_size, dim]")
    pages, kv, page, hd = s if n == 4 else s[1:]
    w = 2 if elem else 4
    if hd * w % 16 or hd * w > 512:
        raise ValueError(f"pages' rows must be whole 16-byte units and 512 bytes at most, got {hd * w}")
    if page < 1 or kv < 1:
        raise ValueError("pages must hold at least one row and one head")
    return _page_strides(k_pages, w), _page_strides(v_pages, w), pages, kv, page, hd


def _check_table(table: torch.Tensor, b: int) -> torch.Tensor:
    s = table.shape
    if len(s) != 2 or s[0] != b:
        raise ValueError(f"page_table must be [{b}, pages of the longest], got {tuple(s)}")
    return table if table.dtype is torch.int32 and table.is_contiguous() else _index("page_table", table, s)


@functools.lru_cache(maxsize=256)
def _cached_workspace(device: int, b: int, n: int, h: int, kv: int, hd: int) -> int:
    with torch.cuda.device(device):
        return _lib.lib().rac_attention_cached_workspace(b, n, h, kv, hd)


def attention_cached(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                     lengths: torch.Tensor, counts: torch.Tensor | None = None,
                     tree: torch.Tensor | None = None, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens, q [batch, nodes, heads, dim], over a paged cache, k_pages and v_pages
    [pages, kv_heads, page_size, dim] of q's type.  Cache row r of sequence b lies in page
    page_table[b, r // page_size].  lengths[b] counts its rows, the new ones included: they are the last
    counts[b] (all `nodes` without counts), at most 64, and are in the cache already (cache_append_).

    New row i sees every row before the new ones and, of those, row j where bit j of tree[b, i] (int64
    [batch, nodes]) is set, or j <= i without a tree.  nodes == 1 is the step of a single token.  A row that
    sees nothing gives zeros.  Rows from counts[b] on keep what `out` holds; without `out` they are zeros.
    Cache rows behind lengths[b] may hold anything, and so may a new row's key where a row does not see it; its
    value must be finite (0 times a NaN or an infinity is NaN), or it reaches the other rows of its sequence.  A page
    number outside the cache is not followed: its rows count as hidden, and check_device_errors() raises."""
    qs = q.shape
    if len(qs) != 4:
        raise ValueError("attention_cached: q [batch, nodes, heads, dim] required")
    b, n, h, hd = qs
    if n > MAX_NEW_ROWS:
        raise ValueError(f"attention_cached: at most {MAX_NEW_ROWS} new rows a sequence, got {n}")
    ks = k_pages.shape
    if len(ks) != 4:
        raise ValueError(f"attention_cached: pages [pages, kv_heads, page_size, {hd}] required")
    _check_heads(h, ks[1], hd)
    elem = _elem(q, k_pages, v_pages)
    kst, vst, pages, kv, page, hd_ = _check_pages(k_pages, v_pages, elem, False)
    if hd_ != hd:
        raise ValueError(f"attention_cached: pages [pages, kv_heads, page_size, {hd}] required")
    table = _check_table(page_table, b)
    lens = _index("lengths", lengths, (b,))
    cnt = _index("counts", counts, (b,)) if counts is not None else None
    if tree is not None:
        if tree.dtype is not torch.int64:
            raise ValueError(f"tree must hold int64 masks, got {tree.dtype}")
        tree = _index("tree", tree, (b, n), torch.int64)
    if out is not None:
        _check_out("out", out, qs, q.dtype)
    d = _device(q, k_pages, v_pages, table, lens, cnt, tree, out)
    q, qp, qst = _rows(q, 2 if elem else 4)
    o = _like(q) if out is None else out
    ws_n = _cached_workspace(d, b, n, h, kv, hd)
    ws = q.new_empty(ws_n, dtype=torch.uint8)
    _launch("rac_attention_cached_async", _lib.CACHED_ARGS.pack(
        qp, k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), lens.data_ptr(),
        0 if cnt is None else cnt.data_ptr(), 0 if tree is None else tree.data_ptr(), o.data_ptr(), ws.data_ptr(),
        *qst, *kst, *vst, ws_n, table.shape[1], pages, page, b, n, h, kv, hd, elem, out is None,
        hd ** -0.5 if scale is None else scale), d)
    return o


def cache_append_(k_pages: torch.Tensor, v_pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                  page_table: torch.Tensor, starts: torch.Tensor, cu_seqlens: torch.Tensor) -> None:
    """Writes new rows k, v [tokens, kv_heads, dim] into a cache's pages [pages, kv_heads, page_size, dim], in
    place: row cu_seqlens[b] + i to cache row starts[b] + i of sequence b.  Rows behind the last sequence are
    not written.  A row whose page is outside the cache is skipped, and check_device_errors() raises."""
    s, ps = k.shape, k_pages.shape
    if len(s) != 3 or v.shape != s or len(ps) != 4 or s[1] != ps[1] or s[2] != ps[3]:
        raise ValueError(f"cache_append_: rows {tuple(s)}, {tuple(v.shape)} do not fit pages {tuple(ps)}")
    elem = _elem(k_pages, v_pages, k, v)
    b = starts.numel()
    table, at = _check_table(page_table, b), _index("starts", starts, (b,))
    cu = _index("cu_seqlens", cu_seqlens, (b + 1,))
    kst, vst, pages, kv, page, hd = _check_pages(k_pages, v_pages, elem, False)
    d = _device(k_pages, v_pages, k, v, table, at, cu)
    w = 2 if elem else 4
    k, kp, ks = _rows(k, w)
    v, vp, vs = _rows(v, w)
    _launch("rac_cache_append_async", _lib.CACHE_ARGS.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), kp, vp, table.data_ptr(), at.data_ptr(), cu.data_ptr(), 0, 0, 0, 0,
        0, *kst, 0, *vst, *ks, *vs, s[0], table.shape[1], pages, page, b, 0, 1, kv, hd, elem), d)


def rope_rows(cos_tab: torch.Tensor, sin_tab: torch.Tensor, positions: torch.Tensor):
    """Rows `positions` ([n], int32 or int64) of RoPE tables [rows, dim / 2], as float32: (cos, sin) [n, dim / 2] for
    rope_apply_.  A position outside the tables gives a row of NaN, and check_device_errors() raises."""
    if cos_tab.dim() != 2 or sin_tab.shape != cos_tab.shape:
        raise ValueError(f"rope_rows: tables must be [rows, dim / 2] and alike, got {tuple(cos_tab.shape)} and "
                         f"{tuple(sin_tab.shape)}")
    if positions.dim() != 1 or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"rope_rows: positions must be 1-D and int32 or int64, got {tuple(positions.shape)} of "
                         f"{positions.dtype}")
    elem = _elem(cos_tab, sin_tab)
    d = _device(cos_tab, sin_tab, positions)
    c, s, pos = cos_tab.contiguous(), sin_tab.contiguous(), positions.contiguous()
    out = c.new_empty((2, pos.shape[0], c.shape[1]), dtype=torch.float32)
    args = (c.data_ptr(), s.data_ptr(), elem, pos.data_ptr(), pos.element_size(), pos.shape[0], c.shape[0], c.shape[1],
            out[0].data_ptr(), out[1].data_ptr())
    with torch.cuda.device(d):
        _lib.call("rac_rope_rows_async", *args, _raw_stream(d))
    return out[0], out[1]


def _layered(st: tuple) -> tuple:
    return st if len(st) == 4 else (0, *st)


def cache_copy_pages_(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copies page src[i] to page dst[i] of a cache's pages [[layers,] pages, kv_heads, page_size, dim], in every
    layer.  No page may be a destination twice, or both a source and a destination: the copies run at once.
    Page numbers outside the cache are skipped, and check_device_errors() raises."""
    if src.dim() != 1 or dst.shape != src.shape:
        raise ValueError(f"src and dst must be 1-D and alike, got {tuple(src.shape)} and {tuple(dst.shape)}")
    s, t = _index("src", src, src.shape), _index("dst", dst, src.shape)
    elem = _elem(k_pages, v_pages)
    kst, vst, pages, kv, page, hd = _check_pages(k_pages, v_pages, elem, True)
    d = _device(k_pages, v_pages, s, t)
    layers = k_pages.shape[0] if len(kst) == 4 else 1
    _launch("rac_cache_copy_pages_async", _lib.CACHE_ARGS.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), 0, 0, 0, 0, 0, s.data_ptr(), t.data_ptr(), 0, 0,
        *_layered(kst), *_layered(vst), 0, 0, 0, 0, 0, 0, pages, page, 0, s.shape[0], layers, kv, hd, elem), d)


def cache_compact_(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
                   accepted: torch.Tensor, n_accepted: torch.Tensor) -> None:
    """Moves the accepted nodes of drafted trees together, in place and in every layer of
    [[layers,] pages, kv_heads, page_size, dim]: cache row starts[b] + accepted[b, i] of sequence b to row
    starts[b] + i, for i < n_accepted[b].  accepted is [batch, nodes], at most 64 wide; a sequence's rows are
    all read before the first is written, so the nodes may come in any order.  Sequences that share a page
    must not both move rows in it."""
    b = starts.numel()
    s = accepted.shape
    if len(s) != 2 or s[0] != b or s[1] > MAX_NEW_ROWS:
        raise ValueError(f"accepted must be [{b}, at most {MAX_NEW_ROWS}], got {tuple(s)}")
    table, at = _check_table(page_table, b), _index("starts", starts, (b,))
    acc, n_acc = _index("accepted", accepted, s), _index("n_accepted", n_accepted, (b,))
    elem = _elem(k_pages, v_pages)
    kst, vst, pages, kv, page, hd = _check_pages(k_pages, v_pages, elem, True)
    d = _device(k_pages, v_pages, table, at, acc, n_acc)
    layers = k_pages.shape[0] if len(kst) == 4 else 1
    _launch("rac_cache_compact_async", _lib.CACHE_ARGS.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), 0, 0, table.data_ptr(), at.data_ptr(), 0, 0, 0, acc.data_ptr(),
        n_acc.data_ptr(), *_layered(kst), *_layered(vst), 0, 0, 0, 0, 0, table.shape[1], pages, page, b, s[1], layers,
        kv, hd, elem), d)


def check_device_errors(device=None) -> None:
    """Synchronises the current stream and raises if a bounded device loop gave up."""
    dev = torch.device("cuda") if device is None else torch.device(device)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().rac_check_device_errors(torch.cuda.current_stream().cuda_stream))
