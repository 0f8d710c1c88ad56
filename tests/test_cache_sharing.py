"""RACPagedCache: steps that are out of date, and pages that forks share."""
import pytest
import torch

from rac_b200 import ext
from rac_b200 import rac_torch as R
from rac_b200.cache import RACPagedCache
from test_cache_pages import _consistent, _rows, _write, quiet  # noqa: F401


def cache(pages, page_size=4, layers=1):
    return RACPagedCache(layers, pages, 1, 32, page_size=page_size, device="cpu")


def out_of_date(c, step):
    assert step.stale()
    with pytest.raises(ValueError, match="moved on"):
        step.attend(0, None, None, None)
    with pytest.raises(ValueError, match="latest"):
        c.accept(step, [[0]] * len(step.ids))


def test_a_step_of_the_same_length_is_another_step(quiet):  # noqa: F811
    """Cut back and taken again, a sequence is as long as before on other pages, which may be another's by then."""
    c = cache(6, 8)
    a, b = c.add(), c.add()
    old = c.step([a], 5)
    c.truncate(a, 0)
    c.step([b], 3)
    new = c.step([a], 5)
    assert c.pages(b) == old.page_table[0].tolist() != new.page_table[0].tolist()
    assert not new.stale()
    out_of_date(c, old)
    # Drafted, accepted in part, drafted again to the same length.
    one = c.step([a], 3, parents=[-1, 0, 0])
    c.accept(one, [[0]])
    two = c.step([a], 2)
    assert one.lengths.tolist() == two.lengths.tolist()
    out_of_date(c, one)
    c.truncate(a, c.length(a))                                  # nothing moves
    assert not two.stale()
    both = c.step([a, b], 1)
    out_of_date(c, two)
    c.free(b)
    out_of_date(c, both)
    _consistent(c)


@pytest.mark.parametrize("drafted,kept", [(8, [0, 3]), (8, [1, 2, 6]), (9, [8]), (6, [0, 1, 5])])
def test_accepted_rows_leave_a_fork_as_it_was(quiet, drafted, kept):  # noqa: F811
    """A fork of a sequence that holds drafted rows shares its full pages: those that receive a moved row are copied."""
    c = cache(12, layers=2)
    a = c.add()
    _write(c, c.step([a], 2), 10)
    step = c.step([a], drafted, parents=[-1] * drafted)
    _write(c, step, 100)
    f = c.fork(a)
    before = _rows(c, a)
    c.accept(step, [kept])
    _consistent(c)
    assert _rows(c, f) == before
    assert _rows(c, a) == before[:2] + [100 + x for x in kept]
    # What neither holds any longer is free, what both hold is still shared.
    assert c.pages(a)[0] != c.pages(f)[0] or kept[:2] == [0, 1]
    c.free(f)
    assert _rows(c, a) == before[:2] + [100 + x for x in kept]
    c.free(a)
    assert c.free_pages == 12


def test_accept_that_does_not_fit_changes_nothing(quiet):  # noqa: F811
    c = cache(4)
    a, b = c.add(), c.add()
    step = c.step([a, b], 4, parents=[-1, 0, 0, 0])
    _write(c, step, 50)
    f, g = c.fork(a), c.fork(b)
    c.step([f], 5)                                              # two pages more: none is left
    pages, rows = c.pages(a), [_rows(c, s) for s in (a, b, g)]
    with pytest.raises(RuntimeError, match="free"):
        c.accept(step, [[1], [2]])
    _consistent(c)
    assert c.pages(a) == pages and [_rows(c, s) for s in (a, b, g)] == rows and not step.stale()
    c.accept(step, [[0], [0, 1]])                               # nothing moves: no page is needed
    assert _rows(c, a) == rows[0][:1] and _rows(c, b) == rows[1][:2] and _rows(c, g) == rows[2]


@pytest.mark.parametrize("rows", [3, 4, 6])
def test_no_layer_writes_after_a_fork(quiet, monkeypatch, rows):  # noqa: F811
    """The rows of a layer that is run after a fork would be missing in the fork's copied page, and would be
    written into pages that it shares: the step is refused.  Its rows may still be accepted."""
    ran = []
    monkeypatch.setattr("rac_b200.ext.cache_append_", lambda *a: ran.append(a))
    c = cache(12, layers=2)
    a, b = c.add(), c.add()
    step = c.step([a, b], rows, parents=[-1] * rows)
    _write(c, step, 7)
    c.fork(b)
    with pytest.raises(ValueError, match="forked"):
        step.attend(1, *[c.k.new_zeros(2 * rows, 1, 32)] * 3)
    assert not ran and not step.stale()
    c.accept(step, [[rows - 1], [0]])
    step = c.step([a, b], 1)
    with pytest.raises(ValueError, match="CUDA"):               # runs, as far as it can here
        step.attend(1, *[c.k.new_zeros(2, 1, 32)] * 3)
    assert len(ran) == 1
    _consistent(c)


@pytest.mark.gpu
def test_forks_of_drafted_rows_answer_on(cuda):
    """A fork taken between a drafted tree and its acceptance goes on with the whole tree's rows, its sequence with the
    accepted ones: each as in a packed pass over them.  32-bit sums of at most 256 terms: 1e-5 of the largest value."""
    torch.manual_seed(0)
    blk = R.RACLlamaBlock(128, 4, ff_dim=192, max_seq_len=64, n_kv_heads=2).to(cuda)
    x = torch.randn(26, 128, device=cuda)

    def whole(rows):
        t = x[rows]
        return blk(t, is_causal=True, cu_seqlens=torch.tensor([0, len(rows)], dtype=torch.int32, device=cuda))

    with torch.no_grad():
        c = RACPagedCache(1, 20, 2, 32, page_size=4, device=cuda)
        a = c.add()
        blk(x[:7], is_causal=True, cache=c.step([a], 7))
        step = c.step([a], 12, parents=[-1, 0, 0] + list(range(2, 11)))       # 0, 1 and 0, 2, 3, ... 11
        blk(x[7:19], is_causal=True, cache=step)
        f = c.fork(a)
        held = [c.k[:, c.pages(f)].clone(), c.v[:, c.pages(f)].clone()]
        c.accept(step, [[0, 2, 3, 4, 5, 6]])
        assert torch.equal(c.k[:, c.pages(f)], held[0]) and torch.equal(c.v[:, c.pages(f)], held[1])
        got = blk(x[19:21], is_causal=True, cache=c.step([a], 2))
        want = whole(list(range(8)) + list(range(9, 14)) + [19, 20])[-2:]
        assert (got - want).abs().max() <= 1e-5 * want.abs().max()
        c.free(a)
        c.truncate(f, 8)
        got = blk(x[8:26], is_causal=True, cache=c.step([f], 18))
        want = whole(list(range(26)))[8:]
        assert (got - want).abs().max() <= 1e-5 * want.abs().max()
    ext.check_device_errors(cuda)
    _consistent(c)
