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
