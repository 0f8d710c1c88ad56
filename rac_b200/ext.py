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

import ctypes as C

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


def _elem(*ts: torch.Tensor) -> int:
    dt = ts[0].dtype
    if dt not in _ELEM:
        raise ValueError(f"float32, float16 or bfloat16 tensors required, got {dt}")
    if any(t.dtype != dt for t in ts):
        raise ValueError(f"tensors of one type required, got {[str(t.dtype) for t in ts]}")
    return _ELEM[dt]


def _same_device(*ts: torch.Tensor) -> None:
    _need_cuda(*ts)
    if any(t is not None and t.device != ts[0].device for t in ts):
        raise ValueError("tensors on one device required")


def _fits(t: torch.Tensor) -> bool:
    """Whether the kernels take t as it lies: contiguous last axis, 16-byte aligned base and strides, no axis
    expanded."""
    e = t.element_size()
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
        s > 0 and s * e % 16 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)


def _lay(t: torch.Tensor) -> torch.Tensor:
    return t if _fits(t) else t.clone(memory_format=torch.contiguous_format)


def _strides(*ts_axes) -> "C.Array":
    """Element strides of the given (tensor, axes); 0 for an axis of one place, whose stride may be anything."""
    v = [t.stride(a) if t.shape[a] > 1 else 0 for t, axes in ts_axes for a in axes]
    return (C.c_longlong * len(v))(*v)


def _index(name: str, t: torch.Tensor, shape: tuple, dtype=torch.int32) -> torch.Tensor:
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must hold int32 or int64, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    return t.to(dtype).contiguous()


def _check_heads(heads: int, kv_heads: int, hd: int) -> None:
    if hd not in (32, 64, 128):
        raise ValueError(f"head size 32, 64 or 128 required, got {hd}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"the query heads ({heads}) must be a multiple of the key/value heads ({kv_heads})")


def _check_out(name: str, out: torch.Tensor, shape: tuple, dtype) -> torch.Tensor:
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"{name} must be a contiguous, 16-byte aligned {tuple(shape)} of {dtype}")
    return out


def _check_packed(q, k, v, cu_seqlens):
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("attention_packed: q [tokens, heads, dim] and k, v [tokens, kv_heads, dim] required")
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError(f"attention_packed: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)} differ")
    _check_heads(q.shape[1], k.shape[1], q.shape[2])
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("attention_packed: cu_seqlens must be 1-D and start with 0")
    elem = _elem(q, k, v)
    return elem, _index("cu_seqlens", cu_seqlens, (cu_seqlens.numel(),))


def _workspace(n: int, like: torch.Tensor):
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n > 0 else None


def _scale(scale, hd: int) -> float:
    return hd ** -0.5 if scale is None else float(scale)


def attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     is_causal: bool = True, scale: float | None = None, out: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v within each sequence of a packed batch, on q [tokens, heads, dim] and
    k, v [tokens, kv_heads, dim] (float32, float16 or bfloat16; head h reads key/value head
    h // (heads // kv_heads)).  Sequence i holds rows cu_seqlens[i] .. cu_seqlens[i + 1] - 1; cu_seqlens
    starts with 0 and rises, lengths of 0 are allowed.  It stays on the device: its values are not checked,
    and no values lead outside the tensors.  scale None is dim ** -0.5.

    Rows behind the last sequence keep what `out` holds; without `out` they are zeros.  What lies in another
    sequence, NaN included, reaches no row.  `lse`, a float32 [heads, tokens], receives the logarithm of each
    row's sum, which attention_packed_backward needs."""
    elem, cu = _check_packed(q, k, v, cu_seqlens)
    t, h, hd = q.shape
    if out is not None:
        _check_out("out", out, q.shape, q.dtype)
    if lse is not None:
        _check_out("lse", lse, (h, t), torch.float32)
    _same_device(q, k, v, cu, out, lse)
    q, k, v = _lay(q), _lay(k), _lay(v)
    o = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    with torch.cuda.device(q.device):
        n = cu.numel() - 1
        ws = _workspace(_lib.lib().rac_attention_packed_workspace(t, n, h, k.shape[1], hd, elem, 0), q)
        _lib.call("rac_attention_packed_async", q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  _strides((q, (0, 1)), (k, (0, 1)), (v, (0, 1))), cu.data_ptr(), n, t, h, k.shape[1],
                  hd, elem, int(bool(is_causal)), _scale(scale, hd), o.data_ptr(), _ptr(lse), int(out is None),
                  _ptr(ws), ws.numel() if ws is not None else 0, _stream(q))
    return o


def attention_packed_backward(grad_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                              out: torch.Tensor, lse: torch.Tensor, cu_seqlens: torch.Tensor,
                              is_causal: bool = True, scale: float | None = None):
    """Gradients (dq, dk, dv) of attention_packed from its out and lse; the key/value heads' sum over the
    query heads that read them.  Rows behind the last sequence get zeros.  The same inputs give the same bits."""
    elem, cu = _check_packed(q, k, v, cu_seqlens)
    if grad_out.shape != q.shape:
        raise ValueError(f"grad_out must be {tuple(q.shape)}, got {tuple(grad_out.shape)}")
    _elem(q, grad_out)
    t, h, hd = q.shape
    _check_out("out", out, q.shape, q.dtype)
    _check_out("lse", lse, (h, t), torch.float32)
    _same_device(q, k, v, cu, grad_out, out, lse)
    q, k, v, g = _lay(q), _lay(k), _lay(v), _lay(grad_out)
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = torch.empty_like(k, memory_format=torch.contiguous_format)
    dv = torch.empty_like(v, memory_format=torch.contiguous_format)
    with torch.cuda.device(q.device):
        n = cu.numel() - 1
        ws = _workspace(_lib.lib().rac_attention_packed_workspace(t, n, h, k.shape[1], hd, elem, 1), q)
        _lib.call("rac_attention_packed_backward_async", g.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  _strides((q, (0, 1)), (k, (0, 1)), (v, (0, 1)), (g, (0, 1))), out.data_ptr(), lse.data_ptr(),
                  cu.data_ptr(), n, t, h, k.shape[1], hd, elem, int(bool(is_causal)), _scale(scale, hd),
                  dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(ws), ws.numel() if ws is not None else 0,
                  _stream(q))
    return dq, dk, dv


def _check_pages(k_pages, v_pages, layers: bool):
    """(type, [layers,] pages, kv_heads, page_size, dim) of a cache's two page tensors."""
    want = (4, 5) if layers else (4,)
    if k_pages.dim() not in want or k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must be alike, " + ("[layers, " if layers else "[") +
                         "pages, kv_heads, page_size, dim]")
    e = k_pages.element_size()
    if k_pages.shape[-1] * e % 16 or k_pages.shape[-1] * e > 512:
        raise ValueError(f"pages' rows must be whole 16-byte units and 512 bytes at most, got {k_pages.shape[-1] * e}")
    if k_pages.shape[-2] < 1 or k_pages.shape[-3] < 1:
        raise ValueError("pages must hold at least one row and one head")
    elem = _elem(k_pages, v_pages)
    if not _fits(k_pages) or not _fits(v_pages):
        raise ValueError("pages need a contiguous last axis and 16-byte aligned rows")
    return elem, k_pages.shape[-4], k_pages.shape[-3], k_pages.shape[-2], k_pages.shape[-1]


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
    Cache rows behind lengths[b] may hold anything.  A page number outside the cache is not followed: its rows
    count as hidden, and check_device_errors() raises."""
    if q.dim() != 4:
        raise ValueError("attention_cached: q [batch, nodes, heads, dim] required")
    b, n, h, hd = q.shape
    if n > MAX_NEW_ROWS:
        raise ValueError(f"attention_cached: at most {MAX_NEW_ROWS} new rows a sequence, got {n}")
    if k_pages.dim() != 4 or k_pages.shape[-1] != hd:
        raise ValueError(f"attention_cached: pages [pages, kv_heads, page_size, {hd}] required")
    _check_heads(h, k_pages.shape[1], hd)
    _elem(q, k_pages, v_pages)
    if page_table.dim() != 2 or page_table.shape[0] != b:
        raise ValueError(f"page_table must be [{b}, pages of the longest], got {tuple(page_table.shape)}")
    table = _index("page_table", page_table, page_table.shape)
    lens = _index("lengths", lengths, (b,))
    cnt = _index("counts", counts, (b,)) if counts is not None else None
    if tree is not None and tree.dtype != torch.int64:
        raise ValueError(f"tree must hold int64 masks, got {tree.dtype}")
    tr = _index("tree", tree, (b, n), torch.int64) if tree is not None else None
    elem, pages, kv, page, _ = _check_pages(k_pages, v_pages, False)
    if out is not None:
        _check_out("out", out, q.shape, q.dtype)
    _same_device(q, k_pages, v_pages, table, lens, cnt, tr, out)
    q = _lay(q)
    o = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    with torch.cuda.device(q.device):
        ws = _workspace(_lib.lib().rac_attention_cached_workspace(b, n, h, kv, hd), q)
        _lib.call("rac_attention_cached_async", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                  _strides((q, (0, 1, 2)), (k_pages, (0, 1, 2)), (v_pages, (0, 1, 2))), table.data_ptr(),
                  table.shape[1], pages, page, lens.data_ptr(), _ptr(cnt), _ptr(tr), b, n, h, kv, hd, elem,
                  _scale(scale, hd), o.data_ptr(), int(out is None), _ptr(ws), ws.numel() if ws is not None else 0,
                  _stream(q))
    return o


def _page_strides(k_pages, v_pages, *more):
    """{layer, page, head, row} strides of both tensors, then those of `more`."""
    lead = [x if x.dim() == 5 else x.unsqueeze(0) for x in (k_pages, v_pages)]
    return _strides((lead[0], (0, 1, 2, 3)), (lead[1], (0, 1, 2, 3)), *more)


def cache_append_(k_pages: torch.Tensor, v_pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                  page_table: torch.Tensor, starts: torch.Tensor, cu_seqlens: torch.Tensor) -> None:
    """Writes new rows k, v [tokens, kv_heads, dim] into a cache's pages [pages, kv_heads, page_size, dim], in
    place: row cu_seqlens[b] + i to cache row starts[b] + i of sequence b.  Rows behind the last sequence are
    not written.  A row whose page is outside the cache is skipped, and check_device_errors() raises."""
    if k.dim() != 3 or k.shape != v.shape or k_pages.dim() != 4 or k.shape[1] != k_pages.shape[1] or \
            k.shape[2] != k_pages.shape[3]:
        raise ValueError(f"cache_append_: rows {tuple(k.shape)}, {tuple(v.shape)} do not fit pages {tuple(k_pages.shape)}")
    _elem(k_pages, v_pages, k, v)
    b = starts.numel()
    if page_table.dim() != 2 or page_table.shape[0] != b:
        raise ValueError(f"page_table must be [{b}, pages of the longest], got {tuple(page_table.shape)}")
    table, at = _index("page_table", page_table, page_table.shape), _index("starts", starts, (b,))
    cu = _index("cu_seqlens", cu_seqlens, (b + 1,))
    elem, pages, kv, page, hd = _check_pages(k_pages, v_pages, False)
    _same_device(k_pages, v_pages, k, v, table, at, cu)
    k, v = _lay(k), _lay(v)
    with torch.cuda.device(k_pages.device):
        _lib.call("rac_cache_append_async", k_pages.data_ptr(), v_pages.data_ptr(),
                  _page_strides(k_pages, v_pages, (k, (0, 1)), (v, (0, 1))), k.data_ptr(), v.data_ptr(),
                  table.data_ptr(), table.shape[1], pages, page, at.data_ptr(), cu.data_ptr(), b, k.shape[0], kv, hd,
                  elem, _stream(k_pages))


def cache_copy_pages_(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copies page src[i] to page dst[i] of a cache's pages [[layers,] pages, kv_heads, page_size, dim], in every
    layer.  No page may be a destination twice, or both a source and a destination: the copies run at once.
    Page numbers outside the cache are skipped, and check_device_errors() raises."""
    if src.dim() != 1 or dst.shape != src.shape:
        raise ValueError(f"src and dst must be 1-D and alike, got {tuple(src.shape)} and {tuple(dst.shape)}")
    s, d = _index("src", src, src.shape), _index("dst", dst, src.shape)
    elem, pages, kv, page, hd = _check_pages(k_pages, v_pages, True)
    _same_device(k_pages, v_pages, s, d)
    layers = k_pages.shape[0] if k_pages.dim() == 5 else 1
    with torch.cuda.device(k_pages.device):
        _lib.call("rac_cache_copy_pages_async", k_pages.data_ptr(), v_pages.data_ptr(),
                  _page_strides(k_pages, v_pages), s.data_ptr(), d.data_ptr(), s.numel(), layers, pages, page, kv, hd,
                  elem, _stream(k_pages))


def cache_compact_(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
                   accepted: torch.Tensor, n_accepted: torch.Tensor) -> None:
    """Moves the accepted nodes of drafted trees together, in place and in every layer of
    [[layers,] pages, kv_heads, page_size, dim]: cache row starts[b] + accepted[b, i] of sequence b to row
    starts[b] + i, for i < n_accepted[b].  accepted is [batch, nodes], at most 64 wide; a sequence's rows are
    all read before the first is written, so the nodes may come in any order.  Sequences that share a page
    must not both move rows in it."""
    b = starts.numel()
    if accepted.dim() != 2 or accepted.shape[0] != b or accepted.shape[1] > MAX_NEW_ROWS:
        raise ValueError(f"accepted must be [{b}, at most {MAX_NEW_ROWS}], got {tuple(accepted.shape)}")
    if page_table.dim() != 2 or page_table.shape[0] != b:
        raise ValueError(f"page_table must be [{b}, pages of the longest], got {tuple(page_table.shape)}")
    table, at = _index("page_table", page_table, page_table.shape), _index("starts", starts, (b,))
    acc, n_acc = _index("accepted", accepted, accepted.shape), _index("n_accepted", n_accepted, (b,))
    elem, pages, kv, page, hd = _check_pages(k_pages, v_pages, True)
    _same_device(k_pages, v_pages, table, at, acc, n_acc)
    layers = k_pages.shape[0] if k_pages.dim() == 5 else 1
    with torch.cuda.device(k_pages.device):
        _lib.call("rac_cache_compact_async", k_pages.data_ptr(), v_pages.data_ptr(), _page_strides(k_pages, v_pages),
                  table.data_ptr(), table.shape[1], pages, page, at.data_ptr(), acc.data_ptr(), n_acc.data_ptr(), b,
                  acc.shape[1], layers, kv, hd, elem, _stream(k_pages))


def check_device_errors(device=None) -> None:
    """Synchronises the current stream and raises if a bounded device loop gave up."""
    dev = torch.device("cuda") if device is None else torch.device(device)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().rac_check_device_errors(torch.cuda.current_stream().cuda_stream))
