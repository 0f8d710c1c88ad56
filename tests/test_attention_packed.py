"""Attention over packed sequences: values and gradients against 64 bits, and what is refused."""
import math

import pytest
import torch

import attention_plain as plain
from rac_b200 import ext
from rac_b200 import rac_torch as R

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
gpu = pytest.mark.gpu


def make(lens, h, kv, d, dt, dev, seed=0, rest=0, gain=1.0):
    """q, k, v as views of one fused projection, the output's gradient, cu_seqlens."""
    g = torch.Generator(device=dev).manual_seed(seed)
    t = sum(lens) + rest
    qkv = (torch.randn(t, h + 2 * kv, d, device=dev, generator=g) * gain).to(dt)
    go = torch.randn(t, h, d, device=dev, generator=g).to(dt)
    cu = torch.tensor([0] + lens).cumsum(0).to(device=dev, dtype=torch.int32)
    return qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:], go, cu


def run_all(q, k, v, go, cu, causal, scale, fine=True):
    lse = torch.empty((q.shape[1], q.shape[0]), device=q.device)
    low = torch.full_like(q, math.nan, memory_format=torch.contiguous_format) if fine else None
    out = ext.attention_packed(q, k, v, cu, causal, scale, lse=lse, out_low=low)
    dq, dk, dv = ext.attention_packed_backward(go, q, k, v, out, lse, cu, causal, scale, low)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def check(got, q, k, v, go, lens, causal, scale):
    val, tol = plain.packed(q, k, v, lens, causal, scale, go)
    n = sum(lens)
    for name in ("out", "dq", "dk", "dv"):
        plain.close(got[name], val[name], tol[name], name)
    # The sum of the weights is 32-bit work on 32-bit scores.
    d, longest = q.shape[2], max(lens)
    bound = plain.e32(longest, d) * (1 + val["lse"][:, :n].abs().max() + d ** 0.5)
    assert (got["lse"][:, :n].double() - val["lse"][:, :n]).abs().max() <= bound


SHAPES = [([1], 1, 1, 64), ([77], 4, 2, 128), ([128], 2, 1, 128), ([129], 2, 2, 64), ([256, 1, 64], 4, 1, 64),
          ([0, 3, 0, 0, 200, 65, 0], 6, 2, 32), ([63, 64, 65, 127, 128, 129], 2, 2, 128), ([515], 8, 8, 64),
          ([300, 41], 16, 1, 128), ([1] * 40, 2, 1, 64), ([5] * 70, 3, 3, 32)]


@gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,h,kv,d", SHAPES)
def test_values_and_gradients(cuda, lens, h, kv, d, causal, dt):
    q, k, v, go, cu = make(lens, h, kv, d, dt, cuda)
    scale = d ** -0.5
    check(run_all(q, k, v, go, cu, causal, scale), q, k, v, go, lens, causal, scale)
    check(run_all(q, k, v, go, cu, causal, scale, fine=False), q, k, v, go, lens, causal, scale)


@gpu
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("lens,causal", [([16] * 20, True), ([100, 60], True), ([500, 30], True), ([64, 64], False)])
def test_short_rows_gradients(cuda, dt, lens, causal):
    """With out_low, dS and the result are each rounded once to the type and nothing else is: their squares add
    up to twice one rounding's, that is 1.41 of the rounded exact gradients' error; 1.5 leaves 6 % for the few
    thousand values' own spread.  dv: the weights and the result."""
    q, k, v, go, cu = make(lens, 8, 4, 64, dt, cuda, seed=11)
    got = run_all(q, k, v, go, cu, causal, 0.125)
    val, _ = plain.packed(q, k, v, lens, causal, 0.125, go)
    for name in ("dq", "dk", "dv"):
        once = (val[name].to(dt).double() - val[name]).norm()
        assert (got[name].double() - val[name]).norm() <= 1.5 * once, name


@gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("gain,scale", [(4.0, 0.25), (0.05, 1.0), (1.0, -0.3), (1.0, 0.0)])
def test_scales(cuda, dt, gain, scale):
    """Sharp rows (scores of +-100), flat ones, a negative scale and none."""
    lens = [190, 70]
    q, k, v, go, cu = make(lens, 4, 2, 64, dt, cuda, seed=3, gain=gain)
    got = run_all(q, k, v, go, cu, True, scale)
    val, tol = plain.packed(q if scale >= 0 else -q, k, v, lens, True, abs(scale), go)
    if scale < 0:
        val["dq"] = -val["dq"]
    # A score's own error is 2^-24 of the sum of its products' magnitudes, times the sharpness of the row.
    sharp = 1 + float((q.double().abs().amax() * k.double().abs().amax()) * 64 ** 0.5 * abs(scale))
    for name in ("out", "dq", "dk", "dv"):
        extra = plain.e32(190, 64) * sharp * val[name].abs().amax()
        plain.close(got[name], val[name], tol[name] + extra, name)


@gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_small_gradients_keep_their_digits(cuda, dt):
    """A loss that is a mean hands down gradients of 1e-6: they lose no more digits than large ones."""
    lens = [300, 33]
    q, k, v, go, cu = make(lens, 4, 2, 64, dt, cuda, seed=4)
    small = 2.0 ** -14 if dt == F16 else 2.0 ** -40
    a = run_all(q, k, v, go, cu, True, 0.125)
    if dt == F16:
        go = (go.float() * small).to(dt)      # the products stay within float16's own range
        b = run_all(q, k, v, go, cu, True, 0.125)
        val, tol = plain.packed(q, k, v, lens, True, 0.125, go)
        for name in ("dq", "dk", "dv"):
            # Results below 2^-14 are subnormal: their step is 2^-24 whatever their size.
            plain.close(b[name], val[name], tol[name] + 2.0 ** -24, name)
    else:
        b = run_all(q, k, v, go * small, cu, True, 0.125)
        for name in ("dq", "dk", "dv"):
            assert torch.equal(b[name].double(), a[name].double() * small) or \
                (b[name].double() / small - a[name].double()).abs().max() <= 4 * plain.HALF[dt] * a[name].abs().max()


@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_other_sequences_and_rest_do_not_matter(cuda, dt):
    """NaN and infinities in the rows of another sequence or behind the last one reach no row; rows behind the
    last sequence stay as they were in `out` and have zero gradients."""
    lens, rest = [70, 100, 31], 50
    q, k, v, go, cu = make(lens, 4, 2, 64, dt, cuda, seed=5, rest=rest)
    clean = run_all(q, k, v, go, cu, True, 0.125)
    bad = [x.clone() for x in (q, k, v, go)]
    for x in bad:
        x[70:170] = math.nan
        x[201:] = math.inf
    got = run_all(*bad, cu, True, 0.125)
    for name in ("out", "dq", "dk", "dv"):
        for sl in (slice(0, 70), slice(170, 201)):
            assert torch.equal(got[name][sl], clean[name][sl]), name
        assert (got[name][201:] == 0).all(), name
    out = torch.full_like(q, 7, memory_format=torch.contiguous_format)
    ext.attention_packed(q, k, v, cu, True, 0.125, out=out)
    assert (out[201:] == 7).all()
    assert torch.equal(out[:201], run_all(q, k, v, go, cu, True, 0.125, fine=False)["out"][:201])


@gpu
def test_no_rows(cuda):
    q = torch.empty(0, 4, 64, device=cuda)
    k = torch.empty(0, 2, 64, device=cuda)
    cu = torch.zeros(3, dtype=torch.int32, device=cuda)
    got = run_all(q, k, k, q, cu, True, 1.0)
    assert got["out"].shape == (0, 4, 64) and got["dk"].shape == (0, 2, 64)
    q, k, v, go, _ = make([9], 4, 2, 64, BF16, cuda)
    got = run_all(q, k, v, go, torch.zeros(1, dtype=torch.int32, device=cuda), True, 1.0)
    assert not any(got[n].any() for n in ("out", "dq", "dk", "dv"))


@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_strides(cuda, dt):
    """Head-major rows, a misaligned base, heads that are one head expanded."""
    lens = [130, 61]
    q, k, v, go, cu = make(lens, 4, 2, 64, dt, cuda, seed=6)
    want = run_all(*(x.contiguous() for x in (q, k, v, go)), cu, True, 0.125)
    major = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, go)]

    def shifted(x):
        buf = torch.empty(x.numel() + 1, dtype=dt, device=cuda)
        return buf[1:].view(x.shape).copy_(x)

    for form in (major, [shifted(x) for x in (q, k, v, go)]):
        got = run_all(*form, cu, True, 0.125)
        assert all(torch.equal(got[n], want[n]) for n in want)
    one = k[:, :1].expand(-1, 2, -1)
    got = run_all(q, one, v, go, cu, True, 0.125)
    want = run_all(q, one.contiguous(), v, go, cu, True, 0.125)
    assert all(torch.equal(got[n], want[n]) for n in want)


@gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_repeated_calls_give_the_same_bits(cuda, dt):
    q, k, v, go, cu = make([400, 90], 8, 2, 128, dt, cuda, seed=7)
    a, b = run_all(q, k, v, go, cu, True, 0.1), run_all(q, k, v, go, cu, True, 0.1)
    assert all(torch.equal(a[n], b[n]) for n in a)


@gpu
def test_differentiable(cuda):
    """rac_attention_packed's gradients are those of attention_packed_backward, also for one key/value head
    expanded over the group (its gradient adds up), and match differences."""
    lens = [33, 20]
    q, k, v, go, cu = make(lens, 4, 2, 32, F32, cuda, seed=8)
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    out = R.rac_attention_packed(*leaves, cu)
    out.backward(go)
    want = run_all(q, k, v, go, cu, True, 32 ** -0.5)
    for leaf, n in zip(leaves, ("dq", "dk", "dv")):
        assert torch.equal(leaf.grad, want[n])
    one = k[:, :1].detach().clone().requires_grad_(True)
    R.rac_attention_packed(q, one.expand(-1, 2, -1), v, cu).backward(go)
    full = run_all(q, one.detach().expand(-1, 2, -1), v, go, cu, True, 32 ** -0.5)["dk"]
    assert torch.allclose(one.grad, full.sum(1, keepdim=True), atol=1e-6)
    # Central differences of sum(out * go) along random directions: the third-order term is h^2 / 6, h = 1e-2,
    # on a sum of magnitude 1; 32-bit sums add 1e-5 / h.
    g = torch.Generator(device=cuda).manual_seed(1)
    for i, n in enumerate(("dq", "dk", "dv")):
        ins = [x.clone() for x in (q, k, v)]
        way = torch.randn(ins[i].shape, device=cuda, generator=g)
        way /= way.norm()
        f = []
        for h in (1e-2, -1e-2):
            x = list(ins)
            x[i] = ins[i] + h * way
            f.append((ext.attention_packed(*x, cu).double() * go.double()).sum().item())
        slope = (want[n].double() * way.double()).sum().item()
        assert abs((f[0] - f[1]) / 2e-2 - slope) <= 5e-3 * max(1.0, abs(slope))


@gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_backward_from_autograd(cuda, dt):
    """The engine calls the backward from a thread of its own, which may have used no GPU before."""
    q, k, v, go, cu = make([140, 33], 8, 2, 128, dt, cuda, seed=9)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    got = torch.autograd.grad(R.rac_attention_packed(*leaves, cu, True, 0.1), leaves, go)
    want = run_all(q, k, v, go, cu, True, 0.1)
    assert all(torch.equal(a, want[n]) for a, n in zip(got, ("dq", "dk", "dv")))


@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_gradient_of_a_sum(cuda, dt):
    """out.sum() hands down one expanded value: strides of zero."""
    q, k, v, go, cu = make([70, 20], 4, 2, 64, dt, cuda, seed=10)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = R.rac_attention_packed(*leaves, cu)
    got = torch.autograd.grad(out.sum(), leaves, retain_graph=True)
    want = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_two_streams_at_once(cuda, dt):
    """Calls that overlap on the GPU keep apart: each has its own workspace, barriers and tensor memory."""
    sets = [make([900, 300, 77], 8, 2, 64, dt, cuda, seed=s) for s in (12, 13)]
    want = [run_all(*s[:3], s[3], s[4], True, 0.125) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run_all(*sets[i][:3], sets[i][3], sets[i][4], True, 0.125)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(a[n], b[n]) for n in a)


@gpu
def test_rows_past_32_bits(cuda):
    """The last of 280000 rows of 64 heads of 128, elements past 2^31; the sequences before are short ones, so that
    the work is small."""
    t, h, n = 280000, 64, 40
    q = torch.zeros(t, h, 128, dtype=BF16, device=cuda)
    k, v = (torch.zeros(t, 1, 128, dtype=BF16, device=cuda) for _ in range(2))
    g = torch.Generator(device=cuda).manual_seed(14)
    for x in (q, k, v):
        x[-n:] = torch.randn(x[-n:].shape, device=cuda, generator=g).to(BF16)
    cu = torch.cat([torch.arange(0, t - n, n), torch.tensor([t - n, t])]).to(device=cuda, dtype=torch.int32)
    out = ext.attention_packed(q, k, v, cu)
    val, tol = plain.packed(q[-n:], k[-n:], v[-n:], [n], True, 128 ** -0.5)
    plain.close(out[-n:], val["out"], tol["out"])


@gpu
def test_capture_and_another_stream(cuda):
    """Captured forward and backward replay on new inputs, two graphs that were captured one after the other
    do not disturb each other; a side stream gives the same bits."""
    sets = []
    for seed in (1, 2):
        q, k, v, go, cu = make([200, 57], 4, 2, 64, BF16, cuda, seed=seed)
        sets.append([x.contiguous() for x in (q, k, v, go)] + [cu])
    want = [run_all(*s, True, 0.125) for s in sets]
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_all(*sets[0], True, 0.125)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[0][n]) for n in got)
    for _ in range(2):
        ins = [x.clone() for x in sets[0]]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run_all(*ins, True, 0.125)
        graphs.append((g, ins, outs))
    for i in (0, 1):
        for a, b in zip(graphs[i][1], sets[i]):
            a.copy_(b)
    for g, _, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(graphs[i][2][n], want[i][n]) for n in want[i])


def test_refusals():
    q, k = torch.zeros(4, 4, 64), torch.zeros(4, 2, 64)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    for args, word in [((q[0], k, k, cu), "tokens"), ((q, k[:3], k[:3], cu), "differ"), ((q, k, k[:, :1], cu), "differ"),
                       ((q[:, :3], k, k, cu), "multiple"), ((q[..., :48], k[..., :48], k[..., :48], cu), "head size"),
                       ((q.half(), k, k, cu), "one type"), ((q.double(), k.double(), k.double(), cu), "float32"),
                       ((q, k, k, cu.float()), "int32"), ((q, k, k, cu[None]), "1-D"), ((q, k, k, cu[:0]), "1-D"),
                       ((q, k, k, cu), "CUDA")]:
        with pytest.raises(ValueError, match=word):
            ext.attention_packed(*args)
    lse = torch.zeros(4, 4)
    for args, word in [((q[:3], q, k, k, q, lse, cu), "grad_out"), ((q, q, k, k, q[:3], lse, cu), "out must"),
                       ((q, q, k, k, q, lse[:3], cu), "lse must"), ((q.half(), q, k, k, q, lse, cu), "one type"),
                       ((q, q, k, k, q, lse, cu), "CUDA")]:
        with pytest.raises(ValueError, match=word):
            ext.attention_packed_backward(*args)


def test_c_entry_refuses():
    from rac_b200 import _lib
    L = _lib.lib()

    def fwd(heads=4, kv=2, hd=64, dt=0, tokens=8, q=256, stride=64, name="rac_attention_packed_async"):
        return getattr(L, name)(_lib.PACKED_ARGS.pack(q, 256, 256, 256, 256, 256, 256, 256, 256, 256, 256, 0, *[stride] * 8,
                                                      tokens, 0, 1, heads, kv, hd, dt, 1, 0, 1.0), None)

    for name in ("rac_attention_packed_async", "rac_attention_packed_backward_async"):
        assert fwd(heads=5, name=name) == -2 and fwd(kv=0, name=name) == -2 and fwd(tokens=-1, name=name) == -2
        assert fwd(hd=80, name=name) == -5 and fwd(dt=3, name=name) == -5
        assert fwd(q=0, name=name) == -1 and getattr(L, name)(None, None) == -1
        assert fwd(q=264, name=name) == -5 and fwd(dt=1, stride=66, name=name) == -5
        assert fwd(name=name) == -3                                          # no workspace
        assert fwd(tokens=0, name=name) == 0


# ── in the modules ─────────────────────────────────────────────────────────

def _plain_block(blk, x, lens, causal):
    """RACLlamaBlock over packed sequences, elementary operations in x's type (autograd runs through)."""
    a, hd = blk.attn, blk.attn.d_head

    def norm(m, y):
        return y * torch.rsqrt(y.square().mean(-1, keepdim=True) + m.eps) * m.weight.to(y.dtype)

    def lin(m, y):
        return y @ m.weight.to(y.dtype).T

    qkv = lin(a.qkv, norm(blk.norm1, x)).view(x.shape[0], -1, hd)
    q, k, v = qkv.split([a.n_heads, a.n_kv_heads, a.n_kv_heads], 1)
    outs, at = [], 0
    for n in lens:
        c, s = a.rope.cos_cache[:n, None].to(x.dtype), a.rope.sin_cache[:n, None].to(x.dtype)

        def rot(y):
            y0, y1 = y[..., 0::2], y[..., 1::2]
            return torch.stack([y0 * c - y1 * s, y0 * s + y1 * c], -1).flatten(-2)

        g = a.n_heads // a.n_kv_heads
        qq, kk = rot(q[at:at + n]), rot(k[at:at + n]).repeat_interleave(g, 1)
        z = torch.einsum("ihd,jhd->hij", qq, kk) * a.scale
        if causal:
            z = z.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -math.inf)
        outs.append(torch.einsum("hij,jhd->ihd", z.softmax(-1), v[at:at + n].repeat_interleave(g, 1)))
        at += n
    h = x + lin(a.out_proj, torch.cat(outs).reshape(x.shape[0], -1))
    y = norm(blk.norm2, h)
    if blk.gated:
        return h + lin(blk.ffn.down, torch.nn.functional.silu(lin(blk.ffn.gate, y)) * lin(blk.ffn.up, y))
    return h + lin(blk.ffn.fc2, torch.nn.functional.silu(lin(blk.ffn.fc1, y)))


@gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kv", [1, 2, 4])
def test_block_over_packed_sequences(cuda, kv, gated):
    """Output, and the gradients of the input and of every weight, against the block in 64 bits: 32-bit
    sums of at most 256 terms through a dozen steps, 1e-5 of the largest value."""
    torch.manual_seed(0)
    lens = [17, 1, 40]
    blk = R.RACLlamaBlock(128, 4, ff_dim=192, max_seq_len=64, gated=gated, n_kv_heads=kv).to(cuda)
    x = torch.randn(sum(lens), 128, device=cuda)
    cu = torch.tensor([0] + lens).cumsum(0).to(device=cuda, dtype=torch.int32)
    go = torch.randn_like(x)
    xi = x.clone().requires_grad_(True)
    y = blk(xi, is_causal=True, cu_seqlens=cu)
    y.backward(go)
    xd = x.double().requires_grad_(True)
    params = dict(blk.named_parameters())
    got = {n: p.grad for n, p in params.items()}
    want_y = _plain_block(blk, xd, lens, True)
    grads = torch.autograd.grad(want_y, [xd] + list(params.values()), go.double())
    for name, a, b in [("y", y, want_y), ("x", xi.grad, grads[0])] + [(n, got[n], b) for n, b in zip(params, grads[1:])]:
        assert (a.double() - b).abs().max() <= 1e-5 * b.abs().max() + 1e-6, name
    with torch.no_grad():
        z = blk(x[None], is_causal=True, cu_seqlens=cu)
        assert (z[0].double() - want_y).abs().max() <= 1e-5 * want_y.abs().max()
        # Rectangular input to a block with grouped heads: sequences of one length.
        r = blk(x[:56].view(2, 28, 128), is_causal=True) if kv < 4 else None
    if r is not None:
        w = _plain_block(blk, x[:56].double(), [28, 28], True)
        assert (r.reshape(56, 128).double() - w).abs().max() <= 1e-5 * w.abs().max()


def test_module_refusals():
    with pytest.raises(ValueError, match="multiple"):
        R.RACRoPEAttention(128, 4, n_kv_heads=3)
    a = R.RACRoPEAttention(128, 4, max_seq_len=8, n_kv_heads=2)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    x = torch.zeros(4, 128)
    with pytest.raises(ValueError, match="no mask"):
        a(x, mask=torch.zeros(4, 4), cu_seqlens=cu)
    with pytest.raises(ValueError, match="packed x"):
        a(x.view(2, 2, 128), cu_seqlens=cu)
    with pytest.raises(ValueError, match="max_seqlen"):
        a(torch.zeros(9, 128), cu_seqlens=cu)
    with pytest.raises(ValueError, match="positions"):
        a(x, cu_seqlens=cu, positions=torch.zeros(3))
    with pytest.raises(ValueError, match="dropout"):
        R.RACRoPEAttention(128, 4, dropout=0.5, n_kv_heads=2).train()(x[None])
