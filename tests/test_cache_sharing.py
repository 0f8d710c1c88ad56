"""RACPagedCache: steps that are out of date, and pages that forks share.  The accounts are the host's and need no GPU."""
import pytest

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
