"""Prompts and token-by-token decoding of a small Gemma-shaped decoder with tbf16.PagedCache.

    python examples/paged_decode.py [--batch 8] [--steps 64] [--fp8] [--keep 256]

The prompts go through tbf16.sdpa (F.scaled_dot_product_attention, routed by tbf16.convert) and into the cache; every
decoding step is one captured CUDA graph: linears on the weight-streaming kernels, QK-norm and rotary embedding in one
pass, cache.append, cache.attend. With --keep the cache is cut to that many positions per head whenever it has grown
64 past them, by the attention weight each position has received from the prompt's last 32 tokens (cache.attend on
their queries; sdpa leaves no weights) and from the tokens decoded. Weights are random: the tokens mean nothing.
"""
import argparse
import pathlib
import sys
import time

import torch
import torch.nn.functional as F

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "turing-bf16_b200"))
import tbf16  # noqa: E402
from tbf16 import ops  # noqa: E402


LAST = 32  # queries of a prompt whose attention weights a cut goes by


class Layer(torch.nn.Module):
    """RMSNorm, grouped-query attention with QK-norm and rotary embedding, RMSNorm, GeGLU."""

    def __init__(self, hidden, heads, kv_heads, head_dim, inter):
        super().__init__()
        lin = lambda i, o: torch.nn.Linear(i, o, bias=False)  # noqa: E731
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.q_proj, self.k_proj = lin(hidden, heads * head_dim), lin(hidden, kv_heads * head_dim)
        self.v_proj, self.o_proj = lin(hidden, kv_heads * head_dim), lin(heads * head_dim, hidden)
        self.gate_proj, self.up_proj, self.down_proj = lin(hidden, inter), lin(hidden, inter), lin(inter, hidden)
        for name, n in (("in_norm", hidden), ("ff_norm", hidden), ("q_norm", head_dim), ("k_norm", head_dim)):
            setattr(self, name, torch.nn.Parameter(torch.zeros(n)))

    def qkv(self, x, cos, sin):
        """x (tokens, hidden), one row of cos / sin per token -> q, k, v (tokens, heads, head_dim)."""
        h = ops.rmsnorm(x, self.in_norm)
        q = self.q_proj(h).view(-1, self.heads, self.head_dim)
        k = self.k_proj(h).view(-1, self.kv_heads, self.head_dim)
        v = self.v_proj(h).view(-1, self.kv_heads, self.head_dim)
        return ops.rmsnorm_rope(q, self.q_norm, cos, sin), ops.rmsnorm_rope(k, self.k_norm, cos, sin), v

    def rest(self, x, attention):
        x = x + self.o_proj(attention.reshape(x.shape[0], -1))
        h = ops.rmsnorm(x, self.ff_norm)
        return x + ops.glu_linear(self.gate_proj(h), self.up_proj(h), self.down_proj.weight16, self.down_proj.weight_scale,
                                  act="gelu_tanh")


class Decoder(torch.nn.Module):
    def __init__(self, layers=4, hidden=1024, heads=8, kv_heads=4, head_dim=256, inter=4096, vocab=32000):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, hidden)
        self.layers = torch.nn.ModuleList(Layer(hidden, heads, kv_heads, head_dim, inter) for _ in range(layers))
        self.norm = torch.nn.Parameter(torch.zeros(hidden))
        self.head = torch.nn.Linear(hidden, vocab, bias=False)
        self.head_dim = head_dim

    def rotary(self, positions):
        """cos, sin (tokens, head_dim) of integer positions (tokens,)."""
        f = 10000.0 ** (-torch.arange(0, self.head_dim, 2, device=positions.device) / self.head_dim)
        a = (positions[:, None] * f).repeat(1, 2)
        return a.cos().bfloat16(), a.sin().bfloat16()

    def prompt(self, tokens, lengths, cache):
        """Prompts (B, S), right-padded, of the given lengths: fills the cache, returns the logits of their last
        tokens (B, vocab)."""
        B, S = tokens.shape
        cache.advance(lengths)
        counts = torch.tensor(lengths, dtype=torch.int32, device=tokens.device)
        x = self.embed(tokens).view(B * S, -1)
        cos, sin = self.rotary(torch.arange(S, device=tokens.device).repeat(B))
        for i, layer in enumerate(self.layers):
            q, k, v = (t.view(B, S, -1, self.head_dim).transpose(1, 2) for t in layer.qkv(x, cos, sin))
            cache.append(k, v, i, counts=counts)
            a = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
            if cache.weights is not None:
                # the newest tokens of each prompt, the first rows of T: attend takes as many as a prompt has
                T = min(LAST, S)
                at = (counts - counts.clamp(max=T))[:, None] + torch.arange(T, device=x.device)
                last = q.transpose(1, 2)[torch.arange(B, device=x.device)[:, None], at.clamp(max=S - 1)]
                cache.attend(last.transpose(1, 2), i)
            x = layer.rest(x, a.transpose(1, 2).reshape(B * S, -1))
        last = x.view(B, S, -1)[torch.arange(B, device=x.device), (counts - 1).long()]
        return self.head(ops.rmsnorm(last, self.norm))

    def step(self, tokens, positions, cache):
        """One new token of every sequence (B,), at the given positions (B,), which the cache has room for
        (cache.advance(1)): logits (B, vocab)."""
        B = tokens.shape[0]
        x = self.embed(tokens)
        cos, sin = self.rotary(positions)
        for i, layer in enumerate(self.layers):
            q, k, v = (t.view(B, -1, 1, self.head_dim) for t in layer.qkv(x, cos, sin))
            cache.append(k, v, i)
            x = layer.rest(x, cache.attend(q, i))
        return self.head(ops.rmsnorm(x, self.norm))


@torch.no_grad()
def generate(model, prompts, steps, dtype=torch.bfloat16, keep=None, page_size=64):
    """Greedy tokens (B, steps) after the prompts (a list of 1-D int64 tensors), and seconds per step."""
    dev, B = prompts[0].device, len(prompts)
    lengths = [len(p) for p in prompts]
    first = model.layers[0]
    cache = tbf16.PagedCache(B, first.kv_heads, model.head_dim, max(lengths) + steps, layers=len(model.layers), dtype=dtype,
                             page_size=page_size, track=keep is not None, device=dev)
    padded = torch.nn.utils.rnn.pad_sequence(prompts, batch_first=True)
    token = model.prompt(padded, lengths, cache).argmax(-1)
    positions = torch.tensor(lengths, device=dev)
    out = [token.clone()]
    # the step as a graph; the run before the capture settles every buffer and writes the rows that the first replay
    # writes again
    cache.advance(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        weights = None if keep is None else cache.weights.clone()
        model.step(token, positions, cache)
        if keep is not None:
            cache.weights.copy_(weights)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token.copy_(model.step(token, positions, cache).argmax(-1))
        positions += 1
    torch.cuda.synchronize()
    t = time.perf_counter()
    for i in range(steps - 1):
        if i:
            if keep is not None and max(cache.lengths) >= keep + 64:
                cache.evict(keep, recent=min(keep, 32))
            cache.advance(1)
        graph.replay()
        out.append(token.clone())
    torch.cuda.synchronize()
    return torch.stack(out, 1), (time.perf_counter() - t) / max(1, steps - 1)


def build(seed=0, **sizes):
    """A converted decoder with random weights on the GPU."""
    torch.manual_seed(seed)
    model = Decoder(**sizes).bfloat16().cuda().eval()
    tbf16.convert(model)
    return model


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--prompt", type=int, default=300, help="longest prompt; the others are shorter")
    ap.add_argument("--fp8", action="store_true", help="8-bit cache")
    ap.add_argument("--keep", type=int, help="positions kept per head")
    args = ap.parse_args()
    model = build()
    prompts = [torch.randint(0, 32000, (max(16, args.prompt - 23 * i),), device="cuda") for i in range(args.batch)]
    tokens, s = generate(model, prompts, args.steps, torch.float8_e4m3fn if args.fp8 else torch.bfloat16, args.keep)
    print(f"{args.batch} sequences, {args.steps} tokens each: {s * 1e6:.0f} us a step, {args.batch / s:.0f} tokens/s")
    print(tokens[:, :8].tolist())


if __name__ == "__main__":
    main()
