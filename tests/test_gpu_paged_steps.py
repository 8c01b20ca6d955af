"""tbf16.PagedCache as a serving loop uses it: what the calls after `advance` take for granted, refused drafts,
steps that were captured, more than one GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rows(B, H, T, D, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(B, h, T, D, device=DEV, generator=g).bfloat16() for h in (H, H, 2 * H)]


def _counts(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _same(a, b):
    for name in ("k", "v", "pos", "weights", "lens", "seen"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name


@pytest.mark.parametrize("T", [3, 5])
def test_calls_take_the_counts_of_the_last_advance(T):
    """A sequence whose count is below T gets its first rows, into the places that advance made, and keeps the tokens
    it had; one without new tokens is left alone. With counts given, the calls do the same as before."""
    import tbf16
    from tbf16 import _ext
    a, b = (tbf16.PagedCache(3, 2, 64, 100, page_size=16, track=True) for _ in range(2))
    k, v, q = _rows(3, 2, 20, 64)
    for c in (a, b):
        c.advance([20, 15, 7])
        c.append(k, v, counts=_counts([20, 15, 7]))
        c.attend(q[:, :, :1], counts=_counts([1, 1, 1]))
    for step, new in enumerate(([3, 1, 0], [0, 2, 3], [1, 1, 1])):
        k, v, q = _rows(3, 2, T, 64, seed=step + 1)
        for c in (a, b):
            c.advance(new)
        a.append(k, v)
        b.append(k, v, counts=_counts(new))
        assert torch.equal(a.attend(q), b.attend(q, counts=_counts(new)))
        _same(a, b)
    assert _ext.device_status() == 0


def test_fewer_query_rows_than_new_tokens():
    """After a prompt, attention of its last tokens alone: the newest T of each."""
    import tbf16
    from tbf16 import _ext
    c = tbf16.PagedCache(2, 2, 64, 100, page_size=16)
    k, v, q = _rows(2, 2, 30, 64)
    c.advance([30, 9])
    c.append(k, v)
    every = c.attend(q, counts=_counts([30, 9]))
    for T in (1, 2):
        last = torch.stack([q[b, :, n - T:n] for b, n in enumerate((30, 9))])
        got = c.attend(last)
        for b, n in enumerate((30, 9)):
            assert torch.equal(got[b], every[b, :, n - T:n])
    c.release(0)
    assert not c.attend(q[:, :, :1])[0].any()
    assert _ext.device_status() == 0


def test_a_captured_step_follows_the_counts_of_advance():
    import tbf16
    a, b = (tbf16.PagedCache(2, 2, 64, 100, page_size=16, track=True) for _ in range(2))
    k, v, q = _rows(2, 2, 4, 64)
    for c in (a, b):
        c.advance(4)
        c.append(k, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.append(k, v)
        out = a.attend(q)
    for i, new in enumerate(([4, 1], [0, 3], [2, 2], [1, 0])):
        for x, y in zip((k, v, q), _rows(2, 2, 4, 64, seed=i + 5)):
            x.copy_(y)
        a.advance(new)
        graph.replay()
        b.advance(new)
        b.append(k, v, counts=_counts(new))
        assert torch.equal(out, b.attend(q, counts=_counts(new)))
        _same(a, b)


def _attend_and_cut(dev):
    import tbf16
    c = tbf16.PagedCache(1, 80, 64, 18000, track=True, device=dev)
    g = torch.Generator().manual_seed(1)
    k, v, q = (torch.randn(1, h, 17000, 64, generator=g).bfloat16().to(dev) for h in (80, 80, 80))
    c.advance(17000)
    c.append(k, v)
    return c.attend(q[:, :, -1:]).cpu(), *(x.cpu() for x in c.compact(16000))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="two GPUs")
def test_every_gpu_of_a_process():
    """Kernels that need more shared memory than a launch may have by default ask for it on each GPU."""
    assert all(torch.equal(x, y) for x, y in zip(_attend_and_cut("cuda:0"), _attend_and_cut("cuda:1")))


def test_calls_run_with_the_caches_device_current(monkeypatch):
    """Whatever device is current, all that a call asks and does happens on the cache's. (Played here: another device
    is current until the call has made the cache's current.)"""
    import tbf16
    c = tbf16.PagedCache(2, 2, 64, 100, track=True)
    k, v, q = _rows(2, 2, 5, 64)
    c.advance(5)
    depth, seen = [0], []

    class Current:
        def __init__(self, device):
            assert torch.device(device) == c.device

        def __enter__(self):
            depth[0] += 1

        def __exit__(self, *exc):
            depth[0] -= 1

    def noting(fn):
        def call(*args):
            seen.append(depth[0] > 0)
            return fn(*args)
        return call

    class Library:
        def __getattr__(self, name):
            return noting(getattr(tbf16.paged.lib(), name))
    c._lib = Library()
    monkeypatch.setattr(torch.cuda, "device", Current)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: c.device.index if depth[0] else c.device.index + 1)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", noting(torch._C._cuda_isCurrentStreamCapturing))
    c.append(k, v)
    c.attend(q)
    c.compact(3)
    assert len(seen) >= 6 and all(seen)


def test_rows_of_any_layout_with_a_padded_head_dim():
    """A head dim that is no multiple of 8, with heads or tokens innermost in memory."""
    import tbf16
    for d in (20, 36, 80):
        k, v, q = _rows(2, 4, 5, d)
        a, b = (tbf16.PagedCache(2, 4, d, 50, page_size=16) for _ in range(2))
        for c, lay in ((a, lambda x: x.contiguous()), (b, lambda x: x.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2))):
            c.advance(5)
            c.append(lay(k), lay(v))
            c.out = c.attend(lay(q)), c.attend(lay(q)[:, :, :1].transpose(2, 3).contiguous().transpose(2, 3))
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and all(torch.equal(x, y) for x, y in zip(a.out, b.out))


def test_advance_is_refused_inside_a_capture():
    """The lengths are the host's: a recorded upload would put the same ones back with every replay."""
    import tbf16
    c = tbf16.PagedCache(2, 2, 64, 100, page_size=16, track=True)
    c.advance(5)
    x, graph = torch.zeros(4, device=DEV), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        for fn in (lambda: c.advance(1), lambda: c.release(0), lambda: c.evict(3)):
            with pytest.raises(RuntimeError):
                fn()
    assert c.lengths == [5, 5] and c.pool.seen == [5, 5]
    c.advance(1)
    assert c.lens.tolist() == [6, 6]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_drafts_that_were_not_accepted(dtype):
    """After a rewind the cache goes on as one that never had those tokens: rows, numbers and lengths, outputs, and the
    weights of the positions that are used again."""
    import tbf16
    from tbf16 import _ext
    kw = dict(layers=2, page_size=16, track=True, dtype=dtype)
    a, b = (tbf16.PagedCache(3, 2, 64, 100, pages=16, **kw) for _ in range(2))
    k, v, q = _rows(3, 2, 30, 64)
    for c in (a, b):
        c.advance([30, 15, 1])
        for layer in range(2):
            c.append(k, v, layer)
            c.attend(q[:, :, :1], layer)
    start = a.weights.clone()
    k, v, q = _rows(3, 2, 4, 64, seed=1)
    accepted = [1, 2, 0]
    a.advance(4)
    for layer in range(2):
        a.append(k, v, layer)
        drafts = a.attend(q, layer)
    a.rewind([4 - c for c in accepted])
    b.advance(accepted)
    for layer in range(2):
        b.append(k, v, layer)
        got = b.attend(q, layer)
    for s, c in enumerate(accepted):
        assert torch.allclose(drafts[s, :, :c].float(), got[s, :, :c].float(), rtol=2.0 ** -7, atol=2.0 ** -7)
    assert a.lengths == b.lengths == [31, 17, 1] and a.lens.tolist() == a.lengths and torch.equal(a.pos, b.pos)
    for s, n in enumerate(a.lengths):
        assert not a.weights[:, s, :, n:].any() and bool((a.weights[:, s, :, :n] >= start[:, s, :, :n]).all())
    a.weights.copy_(b.weights)
    for step in range(20):  # over the positions given back, and into pages that another sequence gave back
        k, v, q = _rows(3, 2, 2 if step == 0 else 1, 64, seed=step + 2)
        outs = []
        for c in (a, b):
            c.advance([1, 1, 2 if step == 0 else 1])
            outs.append([(c.append(k, v, layer), c.attend(q, layer))[1] for layer in range(2)])
        assert all(torch.equal(x, y) for x, y in zip(*outs))
        assert torch.equal(a.weights, b.weights) and torch.equal(a.pos, b.pos) and torch.equal(a.lens, b.lens)
    assert torch.equal(a.seen, b.seen) and sorted(a.pool.free) == sorted(b.pool.free)
    a.evict(20)
    with pytest.raises(RuntimeError):
        a.rewind([1, 0, 0])
    a.advance([2, 0, 0])
    a.rewind([2, 0, 0])
    assert a.lengths == [20, 20, 20] and _ext.device_status() == 0
