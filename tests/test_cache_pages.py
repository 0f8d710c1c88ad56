"""The pages of a key/value cache: rows appended, pages copied, accepted rows moved, and RACPagedCache's accounts."""
import math

import pytest
import torch

from rac_b200 import _lib, ext
from rac_b200 import rac_torch as R
from rac_b200.cache import RACPagedCache, _depths, _masks

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
gpu = pytest.mark.gpu


def pages(layers, n, kv, page, d, dt, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(layers, n, kv, page, d, device=dev, generator=g).to(dt) for _ in range(2)]


@gpu
@pytest.mark.parametrize("dt,d,kv,page", [(F32, 128, 8, 16), (BF16, 64, 1, 24), (F16, 32, 3, 1), (BF16, 128, 2, 64)])
def test_append(cuda, dt, d, kv, page):
    (kp,), (vp,) = pages(1, 40, kv, page, d, dt, cuda)
    lens, starts = [5, 0, 2 * page + 1, 1], [3, 7, 0, page - 1]
    g = torch.Generator(device=cuda).manual_seed(1)
    t = sum(lens) + 2                                         # two rows behind the last sequence
    fused = torch.randn(t, 2 * kv + 1, d, device=cuda, generator=g).to(dt)
    k, v = fused[:, :kv], fused[:, kv:2 * kv]
    table = torch.randperm(40, generator=torch.Generator().manual_seed(2))[:36].view(4, 9).to(torch.int32)
    want = [kp.clone(), vp.clone()]
    at = 0
    for b, (n, s) in enumerate(zip(lens, starts)):
        for i in range(n):
            for w, x in zip(want, (k, v)):
                w[table[b, (s + i) // page], :, (s + i) % page] = x[at + i]
        at += n
    cu = torch.tensor([0] + lens).cumsum(0).to(cuda)
    ext.cache_append_(kp, vp, k, v, table.to(cuda), torch.tensor(starts, device=cuda), cu)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    ext.check_device_errors(cuda)
    # Pages and rows that do not exist: nothing is written, the device reports it.
    bad = table.clone()
    bad[:] = 40
    ext.cache_append_(kp, vp, k, v, bad.to(cuda), torch.tensor(starts, device=cuda), cu)
    with pytest.raises(_lib.RacError):
        ext.check_device_errors(cuda)
    ext.cache_append_(kp, vp, k, v, table.to(cuda), torch.tensor([9 * page, -100, 9 * page, -1], device=cuda),
                      torch.tensor([0, 5, 5, 6, 7], device=cuda))
    with pytest.raises(_lib.RacError):
        ext.check_device_errors(cuda)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


@gpu
@pytest.mark.parametrize("dt,layers,d,kv,page", [(F32, 3, 128, 8, 16), (BF16, 1, 64, 1, 24), (F16, 5, 32, 3, 1)])
def test_copy_pages(cuda, dt, layers, d, kv, page):
    kp, vp = pages(layers, 20, kv, page, d, dt, cuda)
    for form in (lambda x: x, lambda x: x.transpose(2, 3).contiguous().transpose(2, 3)):
        a, b = form(kp.clone()), form(vp.clone())
        src, dst = [3, 0, 3, 19], [7, 8, 1, 18]
        wa, wb = a.clone(), b.clone()
        wa[:, dst], wb[:, dst] = wa[:, src], wb[:, src]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)   # noqa: E731
        ext.cache_copy_pages_(a, b, i32(src), i32(dst))
        assert torch.equal(a, wa) and torch.equal(b, wb)
        ext.cache_copy_pages_(a[0], b[0], i32([5]), i32([6]))
        assert torch.equal(a[0, 6], a[0, 5]) and (layers == 1 or torch.equal(a[1:], wa[1:]))
        ext.cache_copy_pages_(a, b, i32([]), i32([]))
        ext.check_device_errors(cuda)
        wa = a.clone()
        ext.cache_copy_pages_(a, b, i32([20, 2, -1]), i32([2, -3, 4]))
        with pytest.raises(_lib.RacError):
            ext.check_device_errors(cuda)
        assert torch.equal(a, wa)


@gpu
@pytest.mark.parametrize("dt,layers,d,kv,page", [(F32, 2, 128, 8, 16), (BF16, 1, 64, 1, 24), (F16, 3, 32, 3, 1)])
def test_compact(cuda, dt, layers, d, kv, page):
    """Rising nodes whose places overlap the rows they come from, one of them twice, none, all 64."""
    kp, vp = pages(layers, 300, kv, page, d, dt, cuda)
    table = torch.randperm(300, generator=torch.Generator().manual_seed(3)).view(4, 75).to(torch.int32)
    starts = [2, 5, 9, 0]
    lists = [[1, 2, 3, 7, 40], [], [5, 4, 5, 0], list(range(64))]
    acc = torch.tensor([a + [0] * (64 - len(a)) for a in lists], dtype=torch.int32)
    want = [kp.clone(), vp.clone()]
    for b, a in enumerate(lists):
        for w, old in zip(want, (kp, vp)):
            for i, x in enumerate(a):
                r, s = starts[b] + x, starts[b] + i
                w[:, table[b, s // page], :, s % page] = old[:, table[b, r // page], :, r % page]
    n = torch.tensor([len(a) for a in lists], dtype=torch.int32)
    args = [x.to(cuda) for x in (table, torch.tensor(starts), acc, n)]
    ext.cache_compact_(kp, vp, *args)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    ext.check_device_errors(cuda)
    args[2][0, 1] = 64
    args[0][2] = 300
    args[3][3] = -2
    args[3][1] = 1000
    ext.cache_compact_(kp, vp, *args)
    with pytest.raises(_lib.RacError):
        ext.check_device_errors(cuda)


def test_refusals():
    kp = torch.zeros(3, 5, 2, 16, 64)
    i = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 4, dtype=torch.int32)
    rows = torch.zeros(6, 2, 64)
    for call, word in [
            (lambda: ext.cache_copy_pages_(kp, kp[:2], i, i), "alike"), (lambda: ext.cache_copy_pages_(kp, kp, i, i[:1]), "alike"),
            (lambda: ext.cache_copy_pages_(kp, kp, i.float(), i), "src"), (lambda: ext.cache_copy_pages_(kp, kp, i, i), "CUDA"),
            (lambda: ext.cache_copy_pages_(kp[..., :63], kp[..., :63], i, i), "16-byte"),
            (lambda: ext.cache_copy_pages_(kp.transpose(3, 4), kp.transpose(3, 4), i, i), "contiguous last"),
            (lambda: ext.cache_append_(kp[0], kp[0], rows[:, :1], rows[:, :1], table, i, i), "do not fit"),
            (lambda: ext.cache_append_(kp[0], kp[0], rows.half(), rows.half(), table, i, i), "one type"),
            (lambda: ext.cache_append_(kp[0], kp[0], rows, rows, table, i, i), "cu_seqlens"),
            (lambda: ext.cache_append_(kp[0], kp[0], rows, rows, table[:1], i, i), "page_table"),
            (lambda: ext.cache_append_(kp[0], kp[0], rows, rows, table, i, torch.zeros(3, dtype=torch.int32)), "CUDA"),
            (lambda: ext.cache_compact_(kp, kp, table, i, torch.zeros(2, 65, dtype=torch.int32), i), "64"),
            (lambda: ext.cache_compact_(kp, kp, table, i, torch.zeros(1, 4, dtype=torch.int32), i), "accepted"),
            (lambda: ext.cache_compact_(kp, kp, table, i, torch.zeros(2, 4, dtype=torch.int32), i[:1]), "n_accepted"),
            (lambda: ext.cache_compact_(kp, kp, table, i, torch.zeros(2, 4, dtype=torch.int32), i), "CUDA")]:
        with pytest.raises(ValueError, match=word):
            call()


def test_c_entries_refuse():
    L = _lib.lib()

    def call(name, k=256, pages=8, page=16, kv=2, hd=64, dt=0, n=4, layers=1, batch=2, tokens=4, stride=64):
        return getattr(L, name)(_lib.CACHE_ARGS.pack(k, *[256] * 10, *[stride] * 12, tokens, 4, pages, page, batch, n,
                                                     layers, kv, hd, dt), None)

    for name in ("rac_cache_append_async", "rac_cache_copy_pages_async", "rac_cache_compact_async"):
        assert call(name, page=0) == -2 and call(name, kv=0) == -2 and call(name, dt=5) == -2
        assert call(name, k=0) == -1 and getattr(L, name)(None, None) == -1
        assert call(name, k=264) == -5 and call(name, hd=65) == -5 and call(name, stride=65) == -5
    assert call("rac_cache_append_async", tokens=-1) == -2 and call("rac_cache_append_async", tokens=0) == 0
    assert call("rac_cache_copy_pages_async", n=-1) == -2 and call("rac_cache_copy_pages_async", n=0) == 0
    assert call("rac_cache_compact_async", n=65) == -2 and call("rac_cache_compact_async", batch=0) == 0


# ── RACPagedCache: the accounts are the host's and need no GPU ─────────────

@pytest.fixture
def quiet(monkeypatch):
    """Page kernels replaced by their meaning on CPU tensors."""
    def copy(k, v, src, dst):
        for x in (k, v):
            x[:, dst.long()] = x[:, src.long()]

    def compact(k, v, table, starts, acc, n):
        ps = k.shape[-2]
        for b in range(len(n)):
            rows = [int(starts[b]) + int(a) for a in acc[b, :int(n[b])]]
            for x in (k, v):
                got = [x[:, table[b, r // ps], :, r % ps].clone() for r in rows]
                for i, y in enumerate(got):
                    r = int(starts[b]) + i
                    x[:, table[b, r // ps], :, r % ps] = y

    monkeypatch.setattr(ext, "cache_copy_pages_", copy)
    monkeypatch.setattr(ext, "cache_compact_", compact)


def _consistent(c):
    held = [p for s in c._seqs.values() for p in s[0]]
    assert all(c._uses[p] == held.count(p) for p in range(len(c._uses)))
    assert sorted(c._free) == [p for p in range(len(c._uses)) if c._uses[p] == 0]
    assert all(len(p) == -(-n // c.page_size) for p, n in c._seqs.values())


def _write(c, step, seed):
    """Distinct values into a step's new rows, as the layers would; returns them by (sequence, row)."""
    at = 0
    for s, start, n in zip(step.ids, step.starts_host, step.counts_host):
        for i in range(n):
            p = c.pages(s)[(start + i) // c.page_size]
            assert c._uses[p] == 1                        # never a page that another sequence holds
            c.k[:, p, :, (start + i) % c.page_size] = seed + at
            at += 1


def _rows(c, s):
    p = c.pages(s)
    return [c.k[0, p[r // c.page_size], 0, r % c.page_size, 0].item() for r in range(c.length(s))]


def test_cache_accounts(quiet):
    c = RACPagedCache(2, 12, 2, 32, page_size=4, device="cpu")
    a = c.add()
    step = c.step([a], 10)
    assert step.is_prompt and step.tokens == 10 and step.positions.tolist() == list(range(10))
    _write(c, step, 100)
    b = c.fork(a)
    _consistent(c)
    assert c.pages(a)[:2] == c.pages(b)[:2] and c.pages(a)[2] != c.pages(b)[2] and _rows(c, b) == _rows(c, a)
    step = c.step([a, b], 1)
    assert not step.is_prompt and step.lengths.tolist() == [11, 11] and step.starts.tolist() == [10, 10]
    _write(c, step, 200)
    assert _rows(c, a)[:10] == _rows(c, b)[:10] and _rows(c, a)[10] == 200 and _rows(c, b)[10] == 201
    # Back into a page that both hold: it is copied before it is written to.
    c.truncate(a, 6)
    _consistent(c)
    step = c.step([a], 5, parents=[-1, 0, 0, 1, 3])
    assert step.positions.tolist() == [6, 7, 7, 8, 9]
    assert step.tree.tolist() == [[1, 3, 5, 11, 27]]
    _write(c, step, 300)
    before = _rows(c, b)
    c.accept(step, [[0, 2]])
    _consistent(c)
    assert _rows(c, a)[6:] == [300, 302] and _rows(c, b) == before and c.length(a) == 8
    with pytest.raises(ValueError, match="latest"):
        c.accept(step, [[0]])
    assert step.stale()
    c.free(a)
    c.free(b)
    _consistent(c)
    assert c.free_pages == 12


def test_cache_refusals(quiet):
    c = RACPagedCache(1, 3, 1, 32, page_size=4, device="cpu")
    a, b = c.add(), c.add()
    with pytest.raises(RuntimeError, match="free"):
        c.step([a, b], 8)
    assert c.free_pages == 3 and c.length(a) == c.length(b) == 0
    for call, word in [(lambda: c.step([], 1), "at least one"), (lambda: c.step([a, a], 1), "once"),
                       (lambda: c.step([a], 0), "at least one row"), (lambda: c.step([a, b], [1]), "n_new"),
                       (lambda: c.step([7], 1), "no sequence"), (lambda: c.step([a], 2, parents=[-1]), "parent"),
                       (lambda: c.step([a], 2, parents=[-1, 1]), "before it"),
                       (lambda: c.truncate(a, 1), "between"), (lambda: RACPagedCache(1, 1, 1, 80, device="cpu"), "head size"),
                       (lambda: RACPagedCache(1, 1, 1, 64, dtype=torch.int8, device="cpu"), "float32"),
                       (lambda: RACPagedCache(0, 1, 1, 64, device="cpu"), "at least 1")]:
        with pytest.raises(ValueError, match=word):
            call()
    big = RACPagedCache(1, 40, 1, 32, page_size=4, device="cpu")
    s = big.add()
    big.step([s], 70)                                     # a prompt may be longer
    with pytest.raises(ValueError, match="64"):
        big.step([s], 65)
    step = big.step([s], 3)
    with pytest.raises(ValueError, match="rising"):
        big.accept(step, [[1, 0]])
    with pytest.raises(ValueError, match="new rows"):
        big.accept(step, [[3]])
    with pytest.raises(ValueError, match="one list"):
        big.accept(step, [[0], [0]])
    with pytest.raises(ValueError, match="moved on"):
        big.truncate(s, 1)
        step.attend(0, None, None, None)


def test_tree_of_64():
    chain = _masks(list(range(-1, 63)))
    assert chain[0] == 1 and chain[63] == -1 and chain[62] == (1 << 63) - 1
    assert _depths([-1, 0, 0, -1, 2]) == [0, 1, 1, 0, 2]


# ── a model that answers ───────────────────────────────────────────────────

@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_blocks_answer_like_the_whole_prompt(cuda, dt):
    """Two blocks: prompts, single tokens, a fork, a drafted tree with its accepted path, ragged steps.  Each row
    equals the row of the packed pass over the whole sequence: in 32 bits to 1e-5 of the largest value (sums of
    at most 256 terms, two blocks); in bf16 the cache rounds keys and values, 2^-8 each, through two blocks."""
    torch.manual_seed(0)
    blocks = [R.RACLlamaBlock(128, 4, ff_dim=192, max_seq_len=128, n_kv_heads=2).to(cuda) for _ in range(2)]
    g = torch.Generator(device=cuda).manual_seed(1)
    seqs = [torch.randn(n, 128, device=cuda, generator=g) for n in (60, 41)]

    def whole(x):
        cu = torch.tensor([0, x.shape[0]], dtype=torch.int32, device=cuda)
        for b in blocks:
            x = b(x, is_causal=True, cu_seqlens=cu)
        return x

    def step_through(x, step):
        for i, b in enumerate(blocks):
            x = b(x, is_causal=True, cache=step, layer=i)
        return x

    tol = 1e-5 if dt == F32 else 2.0 ** -6

    def same(got, want):
        assert (got - want).abs().max() <= tol * want.abs().max()

    with torch.no_grad():
        want = [whole(x) for x in seqs]
        c = RACPagedCache(2, 40, 2, 32, page_size=16, dtype=dt, device=cuda)
        a, b = c.add(), c.add()
        out = step_through(torch.cat([seqs[0][:30], seqs[1][:17]]), c.step([a, b], [30, 17]))
        same(out, torch.cat([want[0][:30], want[1][:17]]))
        for i in range(3):
            x = torch.stack([seqs[0][30 + i], seqs[1][17 + i]])[:, None]
            out = step_through(x, c.step([a, b], 1))
            same(out[:, 0], torch.stack([want[0][30 + i], want[1][17 + i]]))
        f = c.fork(a)
        # A tree on a: nodes 0, 2, 5 are the true continuation, the others are wrong guesses.
        wrong = torch.randn(3, 128, device=cuda, generator=g)
        t = torch.stack([seqs[0][33], wrong[0], seqs[0][34], wrong[1], wrong[2], seqs[0][35]])
        step = c.step([a], 6, parents=[-1, 0, 0, 1, 2, 2])
        out = step_through(t[None], step)[0]
        same(out[[0, 2, 5]], want[0][33:36])
        c.accept(step, [[0, 2, 5]])
        # A ragged step: seven rows of a behind the accepted ones, two of b, one of the fork.
        step = c.step([a, b, f], [7, 2, 1])
        out = step_through(torch.cat([seqs[0][36:43], seqs[1][20:22], seqs[0][33:34]]), step)
        same(out, torch.cat([want[0][36:43], want[1][20:22], want[0][33:34]]))
        c.free(a)
        x = step_through(seqs[0][34:36], c.step([f], 2))
        same(x, want[0][34:36])
        _consistent(c)
    with pytest.raises(ValueError, match="gradient"):
        step_through(seqs[0][36:37], c.step([f], 1))
    with pytest.raises(ValueError, match="new rows"), torch.no_grad():
        step_through(seqs[0][36:39], c.step([f], 1))
    ext.check_device_errors(cuda)


@gpu
def test_checkpoint_layer_keeps_its_grouped_heads(cuda):
    """load_llama_layer(repeat_kv=False): the same block with a third of the key/value rows."""
    import numpy as np
    from rac_b200 import weights
    rng = np.random.default_rng(0)
    p, d, kvd, ff = "model.layers.0.", 128, 64, 96
    shapes = {"self_attn.q_proj.weight": (d, d), "self_attn.k_proj.weight": (kvd, d),
              "self_attn.v_proj.weight": (kvd, d), "self_attn.o_proj.weight": (d, d),
              "mlp.gate_proj.weight": (ff, d), "mlp.up_proj.weight": (ff, d), "mlp.down_proj.weight": (d, ff),
              "input_layernorm.weight": (d,), "post_attention_layernorm.weight": (d,)}
    t = {p + k: (rng.standard_normal(s) * 0.05 + (len(s) == 1)).astype(np.float32) for k, s in shapes.items()}
    full = weights.load_llama_layer(t, 0, 4, max_seq_len=64, device=cuda)
    kept = weights.load_llama_layer(t, 0, 4, max_seq_len=64, device=cuda, repeat_kv=False)
    assert kept.attn.n_kv_heads == 2 and kept.attn.qkv.out_features == 256
    x = torch.randn(2, 20, d, device=cuda)
    with torch.no_grad():
        a, b = full(x, is_causal=True), kept(x, is_causal=True)
    assert (a - b).abs().max() <= 1e-5 * a.abs().max()
