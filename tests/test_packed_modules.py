"""RACRoPEAttention and RACLlamaBlock beside their grouped heads and packed rows: what is without them, batches without
rows, and 16 bits."""
import copy
import io

import pytest
import torch

from rac_b200 import ext
from rac_b200 import rac_torch as R
from rac_b200.tp import TPLlamaBlock

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
