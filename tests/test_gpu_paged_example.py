"""examples/paged_decode.py: the operators together, as a serving loop uses them."""
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
def _full_logits(model, tokens):
    """Logits at every position of one sequence, recomputed from scratch without the cache."""
    S, d = len(tokens), model.head_dim
    x = model.embed(tokens)
    cos, sin = model.rotary(torch.arange(S, device=tokens.device))
    for layer in model.layers:
        q, k, v = (t.transpose(0, 1).double() for t in layer.qkv(x, cos, sin))
        k, v = (t.repeat_interleave(layer.heads // layer.kv_heads, 0) for t in (k, v))
        s = q @ k.transpose(1, 2) / d ** 0.5
        s = s.masked_fill(torch.ones(S, S, dtype=torch.bool, device=s.device).triu(1), float("-inf"))
        a = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(S, -1).bfloat16()
        x = layer.rest(x, a)
    from tbf16 import ops
    return model.head(ops.rmsnorm(x, model.norm)).float()


@pytest.mark.parametrize("dtype,gap", [(torch.bfloat16, 0.03), (torch.float8_e4m3fn, 0.3)])
def test_decoded_tokens_follow_the_whole_sequence(example, dtype, gap):
    """Every greedy token is the best one of the logits recomputed over the whole sequence, or one whose logit is
    that near to it (bf16 activations differ in their last bits between one row and many; 8-bit rows by 2^-4)."""
    model = example.build(**SIZES)
    prompts = [torch.randint(0, 500, (n,), device="cuda") for n in (70, 17, 33)]
    tokens, _ = example.generate(model, prompts, 24, dtype, page_size=16)
    for p, out in zip(prompts, tokens):
        logits = _full_logits(model, torch.cat([p, out]))[len(p) - 1:-1]
        best = logits.max(-1).values
        chosen = logits.gather(1, out[:, None])[:, 0]
        spread = logits.std()
        assert bool((best - chosen <= gap * spread).all()), ((best - chosen) / spread).max()


def test_cut_cache_decodes_on(example):
    """With a budget per head the loop goes on past it: cuts happen, lengths stay within budget + 64, tokens are valid
    ones, and with a budget that nothing reaches they are those of the uncut cache."""
    model = example.build(**SIZES)
    prompts = [torch.randint(0, 500, (n,), device="cuda") for n in (120, 90)]
    plain, _ = example.generate(model, prompts, 40, page_size=16)
    wide, _ = example.generate(model, prompts, 40, keep=1000, page_size=16)
    assert torch.equal(plain, wide)
    cut, _ = example.generate(model, prompts, 150, keep=64, page_size=16)
    assert cut.shape == (2, 150) and int(cut.min()) >= 0 and int(cut.max()) < 500
    from tbf16 import _ext
    assert _ext.device_status() == 0
