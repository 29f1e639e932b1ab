"""Continuous batching over a paged K/V cache, with rules on the choice.

A small decoder with random weights serves prompts of unlike lengths: each step
takes a chunk of the prompts still being read and one token of every sequence
already decoding, writes their K and V into the pages, attends, and chooses the
next tokens under a repetition penalty and a grammar mask.

    python examples/paged_decode.py [--format f16|q8] [--prompts 12] [--steps 40]
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from malaga_b200.ops import LogitRules, PagedKV, Seqs  # noqa: E402


class Decoder:
    """Embedding, `layers` of attention with a residual, and an LM head (f32 weights, seeded)."""

    def __init__(self, vocab=2000, width=256, layers=2, heads=4, kv_heads=2, seed=0, device="cuda"):
        gen = torch.Generator().manual_seed(seed)
        rand = lambda *s: (torch.randn(*s, generator=gen) / s[-1] ** 0.5).to(device)  # noqa: E731
        self.vocab, self.width, self.layers, self.heads, self.kv_heads = vocab, width, layers, heads, kv_heads
        self.dim = width // heads
        self.embed, self.place = rand(vocab, width) * width ** 0.5, rand(4096, width) * width ** 0.5
        self.qkv = [rand((heads + 2 * kv_heads) * self.dim, width) for _ in range(layers)]
        self.out = [rand(width, width) for _ in range(layers)]
        self.head = 2 * rand(vocab, width)

    def start(self, tokens, positions):
        return self.embed[tokens] + self.place[positions]

    def project(self, layer, x):
        """Queries, keys and values as views of one projection's rows."""
        x = x / x.square().mean(-1, keepdim=True).sqrt()
        y = (x @ self.qkv[layer].to(x.dtype).T).view(len(x), self.heads + 2 * self.kv_heads, self.dim)
        return y.split([self.heads, self.kv_heads, self.kv_heads], dim=1)

    def logits(self, x):
        return x @ self.head.to(x.dtype).T


class Sequence:
    def __init__(self, prompt, pages):
        self.tokens, self.prompt, self.read, self.pages = list(prompt), len(prompt), 0, pages


def serve(model: Decoder, prompts: list[list[int]], steps: int, format="q8", page=16, chunk=32, repetition=1.2,
          allow: torch.Tensor | None = None) -> tuple[list[list[int]], list[list[float]]]:
    """Generates `steps` tokens after every prompt. allow: the grammar's bit row [words] int32, or None.
    Returns the new tokens and their log-probabilities."""
    need = [-(-(len(p) + steps) // page) for p in prompts]
    caches = [PagedKV.empty(sum(need), model.kv_heads, page, model.dim, format) for _ in range(model.layers)]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(1)).tolist()
    seqs = [Sequence(p, [order.pop() for _ in range(n)]) for p, n in zip(prompts, need)]
    scores: list[list[float]] = [[] for _ in prompts]
    while True:
        live = [s for s in seqs if len(s.tokens) < s.prompt + steps]
        if not live:
            return [s.tokens[s.prompt:] for s in seqs], scores
        # the rest of a prompt, a chunk at a time, or the last token
        new = [min(chunk, len(s.tokens) - s.read) for s in live]
        batch = Seqs.of([s.pages for s in live], new, [s.read + n for s, n in zip(live, new)])
        at = [(s, p) for s, n in zip(live, new) for p in range(s.read, s.read + n)]
        x = model.start(torch.tensor([s.tokens[p] for s, p in at], device="cuda"),
                        torch.tensor([p for _, p in at], device="cuda"))
        for layer, cache in enumerate(caches):
            q, k, v = model.project(layer, x)
            cache.write(batch, k, v)
            o = cache.attend(batch, q)
            x = x + o.flatten(1) @ model.out[layer].T
        last = [i - 1 for i in torch.tensor(new).cumsum(0).tolist()]
        said = max(len(s.tokens) for s in live)
        rules = LogitRules(
            history=torch.tensor([s.tokens + [-1] * (said - len(s.tokens)) for s in live], dtype=torch.int32, device="cuda"),
            repetition=torch.full((len(live),), repetition, device="cuda"),
            allow=None if allow is None else allow[None].contiguous())
        ids, logp = rules.choose(model.logits(x[last]).contiguous())
        for s, n, i, score in zip(live, new, ids.tolist(), logp.tolist()):
            s.read += n
            if s.read == len(s.tokens):  # the whole prompt has been read
                s.tokens.append(i)
                scores[seqs.index(s)].append(score)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--format", default="q8", choices=("f16", "q8"))
    ap.add_argument("--prompts", type=int, default=12)
    ap.add_argument("--steps", type=int, default=40)
    args = ap.parse_args()
    model = Decoder()
    gen = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, model.vocab, (int(n),), generator=gen).tolist()
               for n in torch.randint(1, 200, (args.prompts,), generator=gen)]
    bits = torch.rand(-(-model.vocab // 32), 32, generator=gen) < 0.5
    allow = (bits * torch.tensor([1 << i for i in range(31)] + [-(1 << 31)])).sum(-1).to(torch.int32).cuda()
    serve(model, prompts, 2, args.format, allow=allow)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    tokens, scores = serve(model, prompts, args.steps, args.format, allow=allow)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - t0
    for p, t, s in zip(prompts, tokens, scores):
        print(f"{len(p):4d} prompt tokens -> {t[:8]}... mean log-probability {sum(s) / len(s):.3f}")
    print(f"{args.prompts * args.steps / seconds:.0f} tokens/s")


if __name__ == "__main__":
    main()
