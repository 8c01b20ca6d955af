"""The page bookkeeping of tbf16.PagedCache.rewind, which needs no GPU."""
import pytest


def _pool():
    from tbf16.paged import PagePool
    p = PagePool(batch=3, pages=12, page_size=16, max_len=64)
    p.advance([40, 17, 3])
    return p


def test_rewind_gives_back_what_advance_took():
    p = _pool()
    before = list(p.lengths), list(p.seen), [list(o) for o in p.owned], sorted(p.free)
    p.advance([10, 0, 14])
    assert p.fresh == [10, 0, 14]
    p.rewind([10, 0, 14])
    assert before == (p.lengths, p.seen, p.owned, sorted(p.free)) and p.fresh == [0, 0, 0]
    p.advance(4)
    p.rewind([1, 4, 3])
    assert p.lengths == [43, 17, 4] and p.seen == [43, 17, 4] and p.fresh == [3, 0, 1]
    p.rewind([43, 0, 0])
    assert p.lengths == [0, 17, 4] and p.owned[0] == [] and len(p.free) == 9


def test_rewind_refuses_without_change():
    p = _pool()
    p.cut(0, 20)  # as evict does
    p.fixed[0] = 20
    p.advance([2, 0, 0])
    state = lambda: (list(p.lengths), list(p.seen), list(p.fresh), [list(o) for o in p.owned], list(p.free))  # noqa: E731
    before = state()
    for counts in ([3, 0, 0], [0, 18, 0], [0, 0, -1], [1, 1], 4):  # below the cut, too many, negative, wrong number
        with pytest.raises(RuntimeError):
            p.rewind(counts)
        assert state() == before
    p.rewind([2, 0, 0])
    assert p.lengths[0] == 20
