"""Several samples of one image prompt, drawn in parallel from a paged cache.

    python examples/parallel_samples.py [--samples 16] [--steps 12] [--text 300] [--grid 4 24 24]

The KV side of serving n samples of one prompt, with a small random model around it:

1. the prompt (text, then an image's or a clip's patches, then text) is admitted and prefilled:
   per layer, rotary positions on three axes and the cache append in one launch
   (rope.write_paged_kv_batch_rope_axes), then attention over the pool;
2. it is forked into samples that share its blocks (PagedSequences.fork);
3. each decode step appends every sample's token, attends with the shared blocks read once
   for all samples (attention.paged_shared_prefix_attention), and draws the next tokens
   (sampling.sample_tokens) from given random numbers.

A sample's tokens depend on its own random numbers alone: run twice with the same seed, or
with fewer samples, they are the same as long as the model's arithmetic is.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import Tensor

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import augur_b200 as ab  # noqa: E402
from augur_b200.attention import DecodeTables, PrefillQueries, paged_prefill_attention, paged_shared_prefix_attention  # noqa: E402
from augur_b200.rope import RopeAxes, write_paged_kv_batch_rope_axes  # noqa: E402
from augur_b200.sampling import sample_tokens  # noqa: E402
from augur_b200.sequences import PagedSequences  # noqa: E402


class Model:
    """Random projections in the shape of a decoder layer's attention (no MLP), and a random output head."""

    def __init__(self, cfg: ab.QwenConfig, device: torch.device, dtype: torch.dtype, seed: int = 0) -> None:
        g = torch.Generator(device=device).manual_seed(seed)
        heads, kv_heads, dim, hidden = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim, cfg.hidden_size

        def weight(rows: int, cols: int) -> Tensor:
            return (torch.randn(rows, cols, generator=g, device=device) / cols ** 0.5).to(dtype)

        self.cfg, self.heads, self.kv_heads, self.dim = cfg, heads, kv_heads, dim
        self.embed = torch.randn(cfg.vocab_size, hidden, generator=g, device=device).to(dtype)
        self.head = torch.randn(cfg.vocab_size, hidden, generator=g, device=device).to(dtype)
        self.qkv = [weight((heads + 2 * kv_heads) * dim, hidden) for _ in range(cfg.num_hidden_layers)]
        self.o = [weight(hidden, heads * dim) for _ in range(cfg.num_hidden_layers)]
        half = dim // 2
        side = half * 3 // 8
        self.axes = RopeAxes.runs((half - 2 * side, side, side), cfg.rope_theta, device)  # time, height, width

    def forward(self, tokens: Tensor, positions: Tensor, slots: Tensor, pool: ab.PagedKVCache, attend) -> Tensor:
        """Hidden states [tokens, hidden]; attend(layer, q) is the attention over the pool."""
        x = self.embed[tokens]
        for layer in range(self.cfg.num_hidden_layers):
            qkv = (x @ self.qkv[layer].t()).view(len(tokens), -1, self.dim)
            q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
            q = write_paged_kv_batch_rope_axes(pool, q, k, v, slots, positions, self.axes, layer)
            x = x + attend(layer, q).reshape(len(tokens), -1) @ self.o[layer].t()
        return x

    def logits(self, x: Tensor) -> Tensor:
        x = torch.nn.functional.normalize(x.float(), dim=-1).to(x.dtype)
        return (x @ self.head.t()).float() * 3.0


def prompt_positions(text: int, grid: tuple[int, int, int], tail: int, device: torch.device) -> tuple[Tensor, int]:
    """Positions [3, tokens] of text, a grid of patches (time, height, width) and text again, and the next one."""
    t, h, w = grid
    at = torch.arange(t * h * w, device=device)
    patches = torch.stack([at // (h * w), at % (h * w) // w, at % w]) + text
    after = text + max(grid)
    parts = [torch.arange(text, device=device).expand(3, text), patches,
             torch.arange(after, after + tail, device=device).expand(3, tail)]
    return torch.cat(parts, dim=1), after + tail


def generate(samples: int = 16, steps: int = 12, text: int = 300, grid: tuple[int, int, int] = (4, 24, 24), tail: int = 21,
             layers: int = 4, vocab: int = 32003, seed: int = 0, dtype: torch.dtype = torch.bfloat16,
             **settings) -> tuple[Tensor, Tensor]:
    """Tokens [steps, samples] and their logprobs."""
    device = torch.device("cuda", torch.cuda.current_device())
    cfg = ab.QwenConfig(vocab_size=vocab, num_hidden_layers=layers)
    model = Model(cfg, device, dtype)
    n = text + grid[0] * grid[1] * grid[2] + tail
    pool = ab.new_paged_kv_cache(cfg, num_blocks=n // 16 + samples * (steps // 16 + 2) + 8, block_size=16, device=device, dtype=dtype)
    seqs = PagedSequences(pool)
    ids = torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed))
    uniform = torch.rand(steps, samples, generator=torch.Generator().manual_seed(seed + 1)).to(device)
    settings = {"temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.02} | settings

    prompt = seqs.admit(ids.tolist())
    positions, next_position = prompt_positions(text, grid, tail, device)
    tables, queries = DecodeTables([seqs.tables[prompt.seq_id]], device), PrefillQueries([n], device)
    x = model.forward(ids.to(device), positions, torch.from_numpy(prompt.slots).to(device), pool,
                      lambda layer, q: paged_prefill_attention(q, pool, layer, tables, queries))
    batch = [prompt.seq_id, *seqs.fork(prompt.seq_id, samples - 1)]
    x = x[-1:].expand(samples, -1)

    tokens, logprobs = [], []
    for step in range(steps):
        token, logprob = sample_tokens(model.logits(x), uniform[step], **settings)
        tokens.append(token)
        logprobs.append(logprob)
        if step + 1 == steps:
            break
        slots, plan = seqs.shared_prefix_step(batch, cfg.num_attention_heads)
        at = torch.full((3, samples), next_position + step, device=device)
        x = model.forward(token, at, slots, pool, lambda layer, q: paged_shared_prefix_attention(q, pool, layer, plan))
    ab.check_status(device)
    for seq in batch:
        seqs.release(seq)
    return torch.stack(tokens), torch.stack(logprobs)


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--samples", type=int, default=16)
    p.add_argument("--steps", type=int, default=12)
    p.add_argument("--text", type=int, default=300)
    p.add_argument("--grid", type=int, nargs=3, default=(4, 24, 24), metavar=("T", "H", "W"))
    p.add_argument("--seed", type=int, default=0)
    a = p.parse_args()
    tokens, logprobs = generate(a.samples, a.steps, a.text, tuple(a.grid), seed=a.seed)
    for s in range(a.samples):
        print(f"sample {s:3d}  logprob {float(logprobs[:, s].sum()):8.2f}  {tokens[:, s].tolist()}")


if __name__ == "__main__":
    main()
