"""A small serving loop over the 8-bit paged cache.

Random weights, no tokenizer: requests with prompts of different lengths are
served together, prompts in chunks beside requests that already decode.  Every
step is one plan for the batch and, per layer, one fused rotary + quantizing
append and one attention call.

    python examples/kv8_serving.py [--cache e4m3] [--chunk 256] [--new 32]
"""

from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from paged_tierkv_b200 import kv8, ops  # noqa: E402


class Decoder:
    """A transformer's attention path: fused projections, rotary, cache, output."""

    def __init__(self, layers=4, heads=8, kv_heads=2, head_dim=128, vocab=512, blocks=1024, block_size=16,
                 cache_dtype=torch.int8, max_positions=8192, seed=0, device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)
        width = heads * head_dim

        def weight(i, o):
            return (torch.randn(i, o, generator=gen, device=device) * i ** -0.5).to(torch.bfloat16)

        self.heads, self.kv_heads, self.head_dim, self.block_size = heads, kv_heads, head_dim, block_size
        self.embed = weight(vocab, width) * vocab ** 0.5
        self.qkv = [weight(width, (heads + 2 * kv_heads) * head_dim) for _ in range(layers)]
        self.proj = [weight(width, width) for _ in range(layers)]
        self.caches = [kv8.Kv8Cache.allocate(blocks, kv_heads, block_size, head_dim, device, cache_dtype)
                       for _ in range(layers)]
        f = 10000.0 ** (-torch.arange(head_dim // 2, device=device, dtype=torch.float64) * 2 / head_dim)
        angle = torch.arange(max_positions, device=device, dtype=torch.float64)[:, None] * f
        self.rotary = kv8.Rotary(torch.cat([angle.cos(), angle.sin()], 1).float())

    def step(self, tokens, plan, max_q_len):
        """Logits of every packed token of a planned step."""
        x = self.embed[tokens]
        for qkv, proj, cache in zip(self.qkv, self.proj, self.caches):
            h = torch.nn.functional.normalize(x.float(), dim=-1).to(x.dtype) * x.shape[-1] ** 0.5
            y = (h @ qkv).view(len(tokens), -1, self.head_dim)
            q, k, v = y.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
            q = kv8.append(cache, plan, k, v, q=q, positions=plan.positions[:len(tokens)], rotary=self.rotary)
            a = kv8.attention(q, cache, plan, self.head_dim ** -0.5, max_q_len=max_q_len)
            x = x + a.flatten(1) @ proj
        return x.float() @ self.embed.float().t()


def serve(model: Decoder, prompts, new_tokens: int, chunk: int, max_blocks: int = 512):
    """Greedy tokens of every prompt, and the logits each one's last token gave.
    A prompt is fed ``chunk`` tokens a step; a request decodes as soon as its
    prompt is in."""
    n, bs, device = len(prompts), model.block_size, model.embed.device
    plan = kv8.StepPlan.allocate(n, n * chunk, bs, device)
    blocks = model.caches[0].blocks
    table = torch.full((n, max_blocks), -1, dtype=torch.int32, device=device)
    free = torch.arange(blocks, dtype=torch.int32, device=device)
    lens = torch.zeros(n, dtype=torch.int32, device=device)
    count = torch.full((1,), blocks, dtype=torch.int32, device=device)
    fed, out = [0] * n, [[] for _ in range(n)]
    last = [None] * n
    while any(len(o) < new_tokens for o in out):
        take = []
        for r in range(n):
            left = len(prompts[r]) - fed[r]
            take.append(min(chunk, left) if left > 0 else int(len(out[r]) < new_tokens))
        ids = [t for r in range(n) for t in
               (prompts[r][fed[r]:fed[r] + take[r]] if fed[r] < len(prompts[r]) else out[r][-1:][:take[r]])]
        kv8.plan_step(plan, lens, torch.tensor(take, dtype=torch.int32, device=device), table, free, count,
                      tokens=len(ids))
        lens, count = plan.kv_lens, plan.free_count        # the next step's, updated in place
        logits = model.step(torch.tensor(ids, device=device), plan, max(take))
        ends = torch.tensor(take).cumsum(0).tolist()
        best = logits.argmax(-1).tolist()
        for r in range(n):
            fed[r] = min(len(prompts[r]), fed[r] + take[r]) if fed[r] < len(prompts[r]) else fed[r]
            if take[r] and fed[r] == len(prompts[r]) and len(out[r]) < new_tokens:
                out[r].append(best[ends[r] - 1])
                last[r] = logits[ends[r] - 1]
    if ops.read_device_errors():
        raise RuntimeError("a request found no free block, or a table named a block outside the cache")
    return out, last


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--cache", choices=("int8", "e4m3"), default="int8")
    ap.add_argument("--chunk", type=int, default=256)
    ap.add_argument("--new", type=int, default=32)
    args = ap.parse_args()
    model = Decoder(cache_dtype=torch.int8 if args.cache == "int8" else torch.float8_e4m3fn)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 512, (n,), generator=gen).tolist() for n in (1, 17, 300, 1000, 2048)]
    t0 = time.perf_counter()
    out, _ = serve(model, prompts, args.new, args.chunk)
    torch.cuda.synchronize()
    print(f"{sum(map(len, prompts))} prompt and {sum(map(len, out))} new tokens in {time.perf_counter() - t0:.2f} s")
    for p, o in zip(prompts, out):
        print(f"prompt of {len(p)}: {o[:8]} ...")


if __name__ == "__main__":
    main()
