"""Attention of new tokens over a paged cache: values against 64 bits, masks, odd pages, and what is refused."""
import math

import pytest
import torch

import attention_plain as plain
from rac_b200 import _lib, ext

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
gpu = pytest.mark.gpu


def make(lengths, nodes, h, kv, d, page, dt, dev, seed=0, fill=0.0):
    """q, pages (what no sequence holds is `fill`), the table with its pages in any order, lengths."""
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    total = sum(need) + 2
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(need + [1])
    table, at = [], 0
    kp = torch.full((total, kv, page, d), fill, device=dev, dtype=dt)
    vp = kp.clone()
    for n, m in zip(lengths, need):
        mine = order[at:at + m]
        at += m
        table.append(mine + [0] * (width - m))
        for i, p in enumerate(mine):
            r = min(page, n - i * page)
            kp[p, :, :r] = torch.randn(kv, r, d, device=dev, generator=g).to(dt)
            vp[p, :, :r] = torch.randn(kv, r, d, device=dev, generator=g).to(dt)
    q = torch.randn(len(lengths), nodes, h, d, device=dev, generator=g).to(dt)
    return q, kp, vp, torch.tensor(table, dtype=torch.int32, device=dev), \
        torch.tensor(lengths, dtype=torch.int32, device=dev)


def tree_masks(b, nodes, seed):
    """Random trees: every node sees itself and the nodes above it."""
    g = torch.Generator().manual_seed(seed)
    rows = []
    for _ in range(b):
        m = []
        for i in range(nodes):
            up = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            m.append((1 << i) | (m[up] if up >= 0 else 0))
        rows.append([x - (1 << 64) if x >> 63 else x for x in m])
    return torch.tensor(rows, dtype=torch.int64)


SHAPES = [  # lengths, nodes, heads, kv_heads, dim, page
    ([1], 1, 1, 1, 64, 16), ([300], 1, 32, 32, 128, 16), ([17, 0, 513, 64], 1, 8, 2, 128, 64),
    ([100, 7], 7, 4, 1, 32, 24), ([13, 200, 64, 1000], 13, 6, 2, 64, 8), ([64, 400], 64, 8, 2, 128, 64),
    ([65, 129, 511], 33, 4, 4, 64, 1), ([2000], 1, 16, 1, 128, 128), ([1500, 3], 3, 12, 4, 128, 100),
    ([5] * 50, 1, 4, 2, 64, 16), ([4096], 48, 4, 1, 64, 256), ([3000 + 700 * i for i in range(6)], 1, 16, 8, 32, 48)]


@gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("lengths,nodes,h,kv,d,page", SHAPES)
def test_values(cuda, lengths, nodes, h, kv, d, page, dt):
    """A chain and a random tree; what no sequence holds is NaN."""
    q, kp, vp, table, lens = make(lengths, nodes, h, kv, d, page, dt, cuda, fill=math.nan)
    counts = [min(nodes, n) for n in lengths]
    cnt = torch.tensor(counts, dtype=torch.int32, device=cuda)
    for tree in (None, tree_masks(len(lengths), nodes, 5)):
        got = ext.attention_cached(q, kp, vp, table, lens, cnt, None if tree is None else tree.to(cuda), 0.1)
        want, tol = plain.cached(q, kp, vp, table.cpu(), lengths, counts, tree, 0.1)
        plain.close(got, want, tol)
    ext.check_device_errors(cuda)


@gpu
@pytest.mark.parametrize("nodes,dt", [(48, BF16), (32, F16), (16, BF16), (3, F32)])
def test_many_sequences_of_unlike_lengths(cuda, nodes, dt):
    """Blocks whose piece of the work ends anywhere: in a unit's tiles, between units, among empty sequences."""
    lengths = [(0, 1, 2500, 130, 640, 48, 127, 129)[(i * 5) % 8] + (i % 3) for i in range(70)]
    q, kp, vp, table, lens = make(lengths, nodes, 8, 2, 64, 32, dt, cuda, seed=9, fill=math.nan)
    counts = [min(nodes, n) for n in lengths]
    got = ext.attention_cached(q, kp, vp, table, lens, torch.tensor(counts, dtype=torch.int32, device=cuda), None, 0.2)
    want, tol = plain.cached(q, kp, vp, table.cpu(), lengths, counts, None, 0.2)
    plain.close(got, want, tol)
    ext.check_device_errors(cuda)


@gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("nodes,h,dt", [(16, 4, F16), (17, 4, BF16), (32, 8, F16), (64, 8, BF16), (43, 12, F16),
                                        (64, 24, BF16), (33, 24, F32)])
def test_row_counts(cuda, nodes, h, dt, d):
    """Rows of a key/value head (two of them) that fill a half, one, two or more row tiles, or pass them by a few."""
    lengths = [700, nodes, 129, 1]
    q, kp, vp, table, lens = make(lengths, nodes, h, 2, d, 24, dt, cuda, seed=3, fill=math.nan)
    counts = [nodes, nodes, nodes - 1, 1]
    tree = tree_masks(len(lengths), nodes, 7)
    got = ext.attention_cached(q, kp, vp, table, lens, torch.tensor(counts, dtype=torch.int32, device=cuda),
                               tree.to(cuda), 0.1)
    want, tol = plain.cached(q, kp, vp, table.cpu(), lengths, counts, tree, 0.1)
    plain.close(got, want, tol)
    ext.check_device_errors(cuda)


@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_masks(cuda, dt):
    """Rows that see nothing (an empty mask on an empty prefix), a mask that skips the row itself, bits of rows
    that do not exist, all 64 bits; ragged counts keep the rows behind them."""
    lengths, nodes = [64, 6, 70, 3], 64
    q, kp, vp, table, lens = make(lengths, nodes, 4, 2, 64, 16, dt, cuda, fill=math.nan)
    counts = [64, 6, 20, 3]
    tree = torch.full((4, nodes), -1, dtype=torch.int64)
    tree[1, :6] = torch.tensor([0, 1, 2, 0, 63, 32])
    tree[2, :20] = torch.arange(20) * 3
    tree[3, :3] = 0
    cnt = torch.tensor(counts, dtype=torch.int32, device=cuda)
    got = ext.attention_cached(q, kp, vp, table, lens, cnt, tree.to(cuda), 0.125)
    want, tol = plain.cached(q, kp, vp, table.cpu(), lengths, counts, tree, 0.125)
    plain.close(got, want, tol)
    assert (got[1, 0] == 0).all() and (got[1, 3] == 0).all() and (got[3] == 0).all()
    out = torch.full_like(q, 9)
    ext.attention_cached(q, kp, vp, table, lens, cnt, tree.to(cuda), 0.125, out=out)
    for b, n in enumerate(counts):
        assert torch.equal(out[b, :n], got[b, :n]) and (out[b, n:] == 9).all() and (got[b, n:] == 0).all()


@gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_sharp_and_large_scores(cuda, dt):
    """One key takes all the weight; scores beyond exp's range."""
    q, kp, vp, table, lens = make([700], 1, 4, 2, 64, 32, dt, cuda, seed=2)
    kp[table[0, 5].item(), :, 3] = q[0, 0, 0] * 4
    for scale in (1.0, 8.0, -1.0):
        got = ext.attention_cached(q, kp, vp, table, lens, scale=scale)
        want, tol = plain.cached(q, kp, vp, table.cpu(), [700], [1], None, scale)
        # A score's own error: 2^-24 of its products' magnitudes, at most |q| |k| scale, eight roundings' worth.
        size = (q.double().norm(dim=-1).amax() * kp.double().norm(dim=-1).amax() * abs(scale)).item()
        plain.close(got, want, tol + 8 * 2.0 ** -24 * size * vp.double().abs().amax())


@gpu
def test_long_cache_and_pages_in_use_by_two(cuda):
    """Sequences of 20000 and 33 rows that share their first pages; the pages' heads and rows swapped in memory."""
    q, kp, vp, table, lens = make([20000, 33], 2, 8, 2, 128, 64, BF16, cuda, seed=3)
    table[1, 0] = table[0, 0]
    counts = [2, 2]
    got = ext.attention_cached(q, kp, vp, table, lens)
    want, tol = plain.cached(q, kp, vp, table.cpu(), [20000, 33], counts, None, 128 ** -0.5)
    plain.close(got, want, tol)
    swapped = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kp, vp)]
    assert torch.equal(ext.attention_cached(q, *swapped, table, lens), got)
    layered = torch.stack([torch.full_like(kp, math.nan), kp]), torch.stack([torch.full_like(vp, math.nan), vp])
    assert torch.equal(ext.attention_cached(q, layered[0][1], layered[1][1], table, lens), got)


@gpu
def test_pages_past_32_bits(cuda):
    """A page whose first element lies past 2^31 elements of the cache."""
    pages = (1 << 31) // (8 * 64 * 128) + 3
    kp = torch.zeros(pages, 8, 64, 128, dtype=BF16, device=cuda)
    vp = torch.zeros(pages, 8, 64, 128, dtype=BF16, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(0)
    last = pages - 1
    kp[last] = torch.randn(8, 64, 128, device=cuda, generator=g).to(BF16)
    vp[last] = torch.randn(8, 64, 128, device=cuda, generator=g).to(BF16)
    q = torch.randn(1, 1, 8, 128, device=cuda, generator=g).to(BF16)
    table = torch.tensor([[last]], device=cuda)
    lens = torch.tensor([50], device=cuda)
    got = ext.attention_cached(q, kp, vp, table, lens)
    want, tol = plain.cached(q, kp[last:], vp[last:], table.cpu() * 0, [50], [1], None, 128 ** -0.5)
    plain.close(got, want, tol)
    rows = torch.randn(3, 8, 128, device=cuda, generator=g).to(BF16)
    ext.cache_append_(kp, vp, rows, rows, table, lens, torch.tensor([0, 3], device=cuda))
    assert torch.equal(kp[last, :, 50:53], rows.transpose(0, 1))
    ext.cache_copy_pages_(kp, vp, torch.tensor([last], device=cuda), torch.tensor([1], device=cuda))
    assert torch.equal(kp[1], kp[last]) and torch.equal(vp[1], vp[last])


@gpu
def test_bad_pages_are_hidden_and_reported(cuda):
    q, kp, vp, table, lens = make([100, 40], 2, 4, 2, 64, 16, F32, cuda, seed=4)
    table[0, 2] = kp.shape[0]
    table[0, 4] = -7
    got = ext.attention_cached(q, kp, vp, table, lens)
    want, tol = plain.cached(q, kp, vp, table.cpu(), [100, 40], [2, 2], None, 64 ** -0.5)
    plain.close(got, want, tol)
    with pytest.raises(_lib.RacError) as e:
        ext.check_device_errors(cuda)
    assert e.value.status == -6
    ext.check_device_errors(cuda)
    # Lengths beyond the table end at the table; below the new rows, or negative, leave no prefix.
    lens = torch.tensor([10 ** 6, -5], device=cuda)
    assert torch.isfinite(ext.attention_cached(q, kp, vp, table.clamp(0, kp.shape[0] - 1), lens)).all()
    ext.check_device_errors(cuda)


@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_capture_streams_and_repeats(cuda, dt):
    q, kp, vp, table, lens = make([900, 77, 300], 5, 8, 2, 128, 32, dt, cuda, seed=6)
    want = ext.attention_cached(q, kp, vp, table, lens)
    assert torch.equal(ext.attention_cached(q, kp, vp, table, lens), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ext.attention_cached(q, kp, vp, table, lens)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):
        g, qq, ll = torch.cuda.CUDAGraph(), torch.zeros_like(q), torch.ones_like(lens) * 5
        with torch.cuda.graph(g):
            out = ext.attention_cached(qq, kp, vp, table, ll)
        graphs.append((g, qq, ll, out))
    for i, (g, qq, ll, out) in enumerate(graphs):
        qq.copy_(q if i else q * 2)
        ll.copy_(lens)
    for g, *_ in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[1][3], want)
    assert torch.equal(graphs[0][3], ext.attention_cached(q * 2, kp, vp, table, lens))


@gpu
def test_strided_queries(cuda):
    q, kp, vp, table, lens = make([50, 90], 4, 4, 2, 64, 16, BF16, cuda, seed=7)
    want = ext.attention_cached(q, kp, vp, table, lens)
    fused = torch.zeros(2, 4, 8, 64, dtype=BF16, device=cuda)
    fused[:, :, :4] = q
    assert torch.equal(ext.attention_cached(fused[:, :, :4], kp, vp, table, lens), want)
    assert torch.equal(ext.attention_cached(q.transpose(0, 1).contiguous().transpose(0, 1), kp, vp, table, lens), want)
    empty = ext.attention_cached(q[:0], kp, vp, table[:0], lens[:0])
    assert empty.shape == (0, 4, 4, 64)
    none = ext.attention_cached(q, kp, vp, table[:, :0], lens * 0)
    assert not none.any()


def test_refusals():
    q, kp = torch.zeros(2, 3, 4, 64), torch.zeros(5, 2, 16, 64)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    tree = torch.zeros(2, 3, dtype=torch.int64)
    ok = dict(q=q, k_pages=kp, v_pages=kp, page_table=table, lengths=lens)
    for change, word in [({"q": q[0]}, "nodes"), ({"q": torch.zeros(2, 65, 4, 64)}, "64"),
                         ({"k_pages": kp[0]}, "pages"), ({"q": torch.zeros(2, 3, 3, 64)}, "multiple"),
                         ({"q": q[..., :32]}, "pages"), ({"v_pages": kp[:4]}, "alike"), ({"q": q.half()}, "one type"),
                         ({"page_table": table[0]}, "page_table"), ({"page_table": table.float()}, "page_table"),
                         ({"lengths": lens[:1]}, "lengths"), ({"counts": lens.float()}, "counts"),
                         ({"tree": tree.int()}, "int64"), ({"tree": tree[:, :2]}, "tree"),
                         ({"k_pages": kp.transpose(2, 3), "v_pages": kp.transpose(2, 3), "q": torch.zeros(2, 3, 4, 16)},
                          "head size"),
                         ({"out": q[:1]}, "out"), ({}, "CUDA")]:
        with pytest.raises(ValueError, match=word):
            ext.attention_cached(**{**ok, **change})


def test_c_entry_refuses():
    L = _lib.lib()

    def call(q=256, heads=4, kv=2, hd=64, dt=0, nodes=1, batch=1, page=16):
        return L.rac_attention_cached_async(_lib.CACHED_ARGS.pack(
            q, 256, 256, 256, 256, 0, 0, 256, 0, *[64] * 9, 0, 4, 8, page, batch, nodes, heads, kv, hd, dt, 0, 1.0), None)

    assert call(nodes=65) == -2 and call(heads=3) == -2 and call(page=0) == -2 and call(batch=-1) == -2
    assert call(hd=96) == -5 and call(dt=9) == -5 and call(q=264) == -5
    assert call(q=0) == -1 and L.rac_attention_cached_async(None, None) == -1
    assert call(batch=0) == 0 and call(nodes=0) == 0
