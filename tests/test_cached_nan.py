"""NaN in a query over a paged cache: it reaches its own row, and no other."""
import math

import pytest
import torch

from rac_b200 import ext
from test_attention_cached import make

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths,nodes,h,kv,d", [([300, 20], 1, 4, 2, 64), ([900, 33, 70], 7, 8, 2, 128),
                                                  ([3000], 33, 8, 1, 32)])
def test_a_query_of_nan(cuda, lengths, nodes, h, kv, d, dt):
    q, kp, vp, table, lens = make(lengths, nodes, h, kv, d, 16, dt, cuda, seed=5)
    want = ext.attention_cached(q, kp, vp, table, lens)
    assert want.isfinite().all()
    bad = q.clone()
    bad[0, 0, 1, 3] = math.nan
    bad[-1, nodes - 1, h - 1] = math.nan
    got = ext.attention_cached(bad, kp, vp, table, lens)
    hit = bad.isnan().any(-1)
    assert got[hit].isnan().all()
    assert torch.equal(got[~hit], want[~hit])
    ext.check_device_errors(cuda)
