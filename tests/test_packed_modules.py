"""RACRoPEAttention and RACLlamaBlock beside their grouped heads and packed rows: what is without them, batches without
rows, and 16 bits."""
import copy
import io

import pytest
import torch

from rac_b200 import ext
from rac_b200 import rac_torch as R
from rac_b200.cache import RACPagedCache
from rac_b200.tp import TPLlamaBlock
from test_attention_packed import _plain_block

gpu = pytest.mark.gpu


def test_modules_without_grouped_heads_stay_as_they_were():
    """A whole module that was saved before there were key/value heads, and one whose n_heads is set later."""
    blk = R.RACLlamaBlock(64, 4, ff_dim=96, max_seq_len=16)
    for name in ("n_kv_heads", "_kv_heads"):
        blk.attn.__dict__.pop(name, None)
    buf = io.BytesIO()
    torch.save(blk, buf)
    buf.seek(0)
    for old in (torch.load(buf, weights_only=False), copy.deepcopy(blk)):
        assert old.attn.n_kv_heads == 4 and not old.attn._needs_rows(None, None, None)
        assert "n_kv_heads" not in repr(old)
    shard = TPLlamaBlock(R.RACLlamaBlock(64, 4, ff_dim=96, max_seq_len=16), 2, 0).attn
    assert shard.n_kv_heads == shard.n_heads == 2 and "n_kv_heads" not in repr(shard)
    assert not shard._needs_rows(None, None, None)
    kept = copy.deepcopy(R.RACRoPEAttention(64, 4, n_kv_heads=2))
    assert kept.n_kv_heads == 2 and kept._needs_rows(None, None, None)
    kept.n_heads, kept.n_kv_heads = 2, 1                        # a shard of grouped heads
    assert kept.n_kv_heads == 1 and kept._needs_rows(None, None, None)


@gpu
@pytest.mark.parametrize("kv", [2, 4])
def test_block_without_rows(cuda, kv):
    """A packed batch of empty sequences, and rectangular ones of no rows: nothing comes out."""
    blk = R.RACLlamaBlock(128, 4, ff_dim=192, max_seq_len=64, n_kv_heads=kv).to(cuda)
    cu = torch.zeros(3, dtype=torch.int32, device=cuda)
    shapes = [((0, 128), dict(cu_seqlens=cu)), ((1, 0, 128), dict(cu_seqlens=cu))]
    if kv < 4:
        shapes += [((2, 0, 128), {}), ((0, 5, 128), {})]
    for shape, kw in shapes:
        x = torch.zeros(shape, device=cuda)
        with torch.no_grad():
            assert blk(x, is_causal=True, **kw).shape == shape
        assert blk(x, is_causal=True, **kw).shape == shape
    ext.check_device_errors(cuda)


@gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kv", [1, 2, 4])
def test_block_in_16_bits(cuda, kv, gated, dt):
    """Output, and gradients of the input and every weight, against the block in 64 bits, relative to their norms.
    Some 12 tensors between the input and the output are rounded, half a step each (u), and some 24 on the way back:
    independent, they add up to sqrt(12) and sqrt(24) half steps; none changes another's size by more than 2."""
    torch.manual_seed(0)
    lens, u = [17, 1, 40], torch.finfo(dt).eps / 2
    blk = R.RACLlamaBlock(128, 4, ff_dim=192, max_seq_len=64, gated=gated, n_kv_heads=kv, dtype=dt, device=cuda)
    x = torch.randn(sum(lens), 128, device=cuda).to(dt)
    cu = torch.tensor([0] + lens).cumsum(0).to(device=cuda, dtype=torch.int32)
    go = torch.randn_like(x)
    xi = x.clone().requires_grad_(True)
    y = blk(xi, is_causal=True, cu_seqlens=cu)
    y.backward(go)
    xd, params = x.double().requires_grad_(True), dict(blk.named_parameters())
    want = _plain_block(blk, xd, lens, True)
    grads = torch.autograd.grad(want, [xd] + list(params.values()), go.double())
    with torch.no_grad():
        z = blk(x, is_causal=True, cu_seqlens=cu)
        c = RACPagedCache(1, 8, kv, 32, page_size=16, dtype=dt, device=cuda)
        w = blk(x, is_causal=True, cache=c.step([c.add() for _ in lens], lens))
    for name, a, b, n in [("y", y, want, 12), ("inference", z, want, 12), ("into a cache", w, want, 12),
                          ("x", xi.grad, grads[0], 24)] + \
            [(m, p.grad, g, 24) for (m, p), g in zip(params.items(), grads[1:])]:
        assert a.dtype == dt
        assert (a.double() - b).norm() <= 2 * n ** 0.5 * u * b.norm(), name
