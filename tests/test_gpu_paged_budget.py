"""examples/paged_decode.py with a budget: what its cuts go by, that they happen, and that captured steps go on over
the cut cache."""
import pathlib
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "examples"))
SIZES = dict(layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, inter=512, vocab=500)


@pytest.fixture(scope="module")
def example():
    import paged_decode
    import tbf16
    yield paged_decode
    tbf16.uninstall_sdpa()


@torch.no_grad()
def test_a_prompts_last_tokens_start_the_totals(example):
    """Every query row adds weights that sum to 1: the group's rows (2) of the last 32 tokens, or of all."""
    import tbf16
    model = example.build(**SIZES)
    lengths = [70, 17, 40]
    cache = tbf16.PagedCache(3, 2, 64, 100, layers=2, page_size=16, track=True)
    tokens = torch.randint(0, 500, (3, 70), device="cuda")
    model.prompt(tokens, lengths, cache)
    for b, n in enumerate(lengths):
        w = cache.weights[:, b]
        assert bool((w[..., :n] > 0).all()) and not w[..., n:].any()
        want = 2.0 * min(32, n)
        assert bool(((w.sum(-1) - want).abs() <= want * 2.0 ** -15).all())


def test_cuts_happen_and_keep_to_the_budget(example, monkeypatch):
    """150 tokens past a budget of 64: the cache is cut whenever it has grown 64 past it, to the budget, and never
    holds more; a budget that nothing reaches cuts nothing."""
    import tbf16
    cuts, most = [], [0]
    evict, advance = tbf16.PagedCache.evict, tbf16.PagedCache.advance

    def noted_evict(self, keep, recent=0):
        before = self.lengths
        weights, pos, seen = self.weights.clone(), self.pos.clone(), self.seen.tolist()
        evict(self, keep, recent)
        cuts.append((before, self.lengths))
        for b, n in enumerate(before):
            m = min(n, keep)
            for layer in range(2):
                for h in range(2):
                    rank = sorted(range(n), key=lambda i: (int(pos[layer, b, h, i]) < seen[b] - recent,
                                                           -float(weights[layer, b, h, i]), i))[:m]
                    assert sorted(self.pos[layer, b, h, :m].tolist()) == sorted(int(pos[layer, b, h, i]) for i in rank)

    def noted_advance(self, counts):
        advance(self, counts)
        most[0] = max(most[0], *self.lengths)
    monkeypatch.setattr(tbf16.PagedCache, "evict", noted_evict)
    monkeypatch.setattr(tbf16.PagedCache, "advance", noted_advance)
    model = example.build(**SIZES)
    prompts = [torch.randint(0, 500, (n,), device="cuda") for n in (120, 90)]
    example.generate(model, prompts, 20, keep=1000, page_size=16)
    assert not cuts
    most[0] = 0
    example.generate(model, prompts, 150, keep=64, page_size=16)
    # 120 tokens, 1 before the loop: cut at 128, then each time 64 more are there
    assert [c[0][0] for c in cuts] == [128] * 3 and all(x <= 64 for _, after in cuts for x in after)
    assert most[0] == 128


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_a_captured_step_goes_on_after_a_cut(dtype):
    """A step captured before any cut, replayed over caches that have been cut, against eager calls on a cache that has
    been cut the same."""
    import tbf16
    B, H, D, L = 2, 2, 64, 2
    a, b = (tbf16.PagedCache(B, H, D, 200, layers=L, page_size=16, track=True, dtype=dtype) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v, q = (torch.randn(B, h, 1, D, device="cuda", generator=g).bfloat16() for h in (H, H, 4))
    prompt = torch.randn(2, B, H, 90, D, device="cuda", generator=g).bfloat16()
    for c in (a, b):
        c.advance([90, 55])
        for layer in range(L):
            c.append(*prompt, layer)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = []
        for layer in range(L):
            a.append(k, v, layer)
            outs.append(a.attend(q, layer))
    for step in range(60):
        for x in (k, v, q):
            x.normal_(generator=g)
        if step in (5, 30):
            for c in (a, b):
                c.evict(40, recent=10)
            assert a.lengths == [40, 40]
        a.advance(1)
        graph.replay()
        b.advance(1)
        for layer in range(L):
            b.append(k, v, layer)
            assert torch.equal(outs[layer], b.attend(q, layer))
        assert torch.equal(a.weights, b.weights) and torch.equal(a.pos, b.pos)
