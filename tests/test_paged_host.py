"""The page bookkeeping of tbf16.PagedCache and its refusals that need no GPU."""
import pytest
import torch


def test_pool_takes_and_returns_pages():
    from tbf16.paged import PagePool
    p = PagePool(batch=3, pages=7, page_size=16, max_len=64)
    assert p.advance([1, 16, 17]) and p.lengths == [1, 16, 17] and p.seen == [1, 16, 17]
    assert [len(o) for o in p.owned] == [1, 1, 2] and len(p.free) == 3
    assert not p.advance([15, 0, 15])  # inside the pages it has
    assert p.advance([1, 1, 1]) and p.lengths == [17, 17, 33] and len(p.free) == 0
    held = sorted(x for o in p.owned for x in o) + sorted(p.free)
    assert sorted(held) == list(range(7))  # no page lost, none held twice


def test_pool_refuses_without_change():
    from tbf16.paged import PagePool
    p = PagePool(batch=2, pages=3, page_size=16, max_len=32)
    p.advance([16, 16])
    before = (list(p.lengths), list(p.seen), [list(o) for o in p.owned], list(p.free))
    for counts in ([1, 1], [17, 0], [-1, 0], [1, 1, 1]):  # pages, max_len, negative, wrong number
        with pytest.raises(RuntimeError):
            p.advance(counts)
        assert before == (list(p.lengths), list(p.seen), [list(o) for o in p.owned], list(p.free))


def test_pool_cut_frees_whole_pages_only():
    from tbf16.paged import PagePool
    p = PagePool(batch=1, pages=4, page_size=16, max_len=64)
    p.advance(50)
    own = list(p.owned[0])
    p.cut(0, 33)
    assert p.lengths == [33] and p.owned[0] == own[:3] and p.seen == [50]
    p.cut(0, 40)  # never longer
    assert p.lengths == [33]
    assert p.rows(4) == [own[:3] + [0]]
    p.cut(0, 0)
    assert sorted(p.free) == [0, 1, 2, 3] and p.rows(4) == [[0, 0, 0, 0]]


def test_cache_refuses_cpu_tensors_and_bad_arguments():
    import tbf16
    with pytest.raises(RuntimeError):
        tbf16.PagedCache(1, 2, 64, 128, device="cpu")
    for bad in (dict(head_dim=257), dict(batch=0), dict(dtype=torch.float16), dict(max_len=0)):
        kw = dict(batch=1, kv_heads=2, head_dim=64, max_len=128, device="cpu") | bad
        with pytest.raises(RuntimeError):
            tbf16.PagedCache(**kw)
