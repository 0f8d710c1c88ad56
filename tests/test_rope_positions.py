"""Positions of packed rows that the RoPE tables do not hold: refused, or reported by the device."""
import pytest
import torch

from rac_b200 import _lib, ext
from rac_b200 import rac_torch as R

gpu = pytest.mark.gpu


def test_rows_past_the_tables_are_refused():
    """Where the host knows the positions it refuses them, before anything runs."""
    a = R.RACRoPEAttention(128, 4, max_seq_len=8, n_kv_heads=2)
    x = torch.zeros(1, 9, 128)
    with pytest.raises(ValueError, match="RoPE tables"):
        a(x)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="RoPE tables"):
        a(x[0], cu_seqlens=cu, max_seqlen=9)
    for bad in (8, -1):
        with pytest.raises(ValueError, match="RoPE tables"):
            a(x[:, :4], positions=torch.tensor([0, 1, bad, 2]))
        with pytest.raises(ValueError, match="RoPE tables"):
            a(x[0, :4], cu_seqlens=cu, positions=torch.tensor([0, 1, bad, 2]))


@gpu
def test_rows_past_the_tables_are_reported(cuda):
    """Where only the device knows the positions, the error word is set, the sequences that the tables hold are as they
    were, and rows behind the last sequence count for nothing."""
    torch.manual_seed(0)
    a = R.RACRoPEAttention(128, 4, max_seq_len=16, n_kv_heads=2).to(cuda)
    x = torch.randn(40, 128, device=cuda)
    cu = torch.tensor([0, 10, 27, 30], dtype=torch.int32, device=cuda)
    with torch.no_grad():
        got = a(x, is_causal=True, cu_seqlens=cu, max_seqlen=16)          # the second has 17 rows
        with pytest.raises(_lib.RacError) as e:
            ext.check_device_errors(cuda)
        assert e.value.status == -6
        ok = torch.tensor([0, 10, 26, 27, 30], dtype=torch.int32, device=cuda)
        want = a(x, is_causal=True, cu_seqlens=ok, max_seqlen=16)
        ext.check_device_errors(cuda)
        assert torch.equal(got[:26], want[:26]) and torch.equal(got[27:], want[27:])
        assert got[26].isnan().all()
        pos = torch.arange(40, device=cuda) % 16
        pos[30:] = torch.tensor([16, -1] * 5, device=cuda)                # behind the last sequence
        a(x, is_causal=True, cu_seqlens=cu, positions=pos)
        ext.check_device_errors(cuda)
        for bad in (16, -1, 1 << 31, -(1 << 40)):
            pos[3] = bad
            got = a(x, is_causal=True, cu_seqlens=cu, positions=pos)
            with pytest.raises(_lib.RacError):
                ext.check_device_errors(cuda)
            assert got[3].isnan().all() and got[10:30].isfinite().all()
            dense = a(x.view(4, 10, 128), positions=pos[:10])
            with pytest.raises(_lib.RacError):
                ext.check_device_errors(cuda)
            assert dense.isnan().any()
    # No row of the tables out of range: gradients as ever.
    xi = x.clone().requires_grad_(True)
    a(xi, is_causal=True, cu_seqlens=ok, max_seqlen=16).sum().backward()
    ext.check_device_errors(cuda)
    assert xi.grad.isfinite().all() and not xi.grad[30:].any()


@gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_table_rows(cuda, dt):
    """The tables' rows at the given positions, in 32 bits, whatever the tables' type and the positions'."""
    g = torch.Generator(device=cuda).manual_seed(1)
    c, s = (torch.randn(33, 16, device=cuda, generator=g).to(dt) for _ in range(2))
    for it in (torch.int32, torch.int64):
        pos = torch.randint(0, 33, (70,), device=cuda, generator=g).to(it)
        got = ext.rope_rows(c, s, pos)
        assert torch.equal(got[0], c[pos.long()].float()) and torch.equal(got[1], s[pos.long()].float())
    assert ext.rope_rows(c, s, pos[:0])[0].shape == (0, 16)
    ext.check_device_errors(cuda)
    for call, word in [((c, s[:3], pos), "alike"), ((c, s, pos.float()), "int"), ((c, s, pos[None]), "1-D"),
                       ((c.double(), s.double(), pos), "float32"), ((c, s, pos.cpu()), "CUDA")]:
        with pytest.raises(ValueError, match=word):
            ext.rope_rows(*call)


def test_c_entry_refuses():
    def call(cos=256, dtype=0, pos=256, width=4, n=3, rows=8, half=16, out=256):
        return _lib.lib().rac_rope_rows_async(cos, 256, dtype, pos, width, n, rows, half, out, 256, None)

    assert call(n=-1) == -2 and call(rows=-1) == -2 and call(half=0) == -2 and call(width=2) == -2
    assert call(dtype=3) == -5 and call(cos=0) == -1 and call(pos=0) == -1 and call(out=0) == -1
    assert call(n=0) == 0
