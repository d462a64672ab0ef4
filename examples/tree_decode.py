"""Decoding with drafted trees over a paged cache, on one GPU.

A toy attention layer (random projections, no training) serves a few requests:
their prompts enter the cache in one step, then each step drafts a tree of
tokens per request, attends all its nodes at once and keeps one root-to-leaf
path. At the end the same tokens run again one by one, and the outputs of the
two ways are compared.

    python examples/tree_decode.py [--requests 4] [--steps 6] [--nodes 13] [--heads 8] [--kv-heads 2] [--dim 64]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch  # noqa: E402

from flashlite_b200.rotary import rotary_table  # noqa: E402
from flashlite_b200.serving import PagedCache  # noqa: E402


class Layer:
    """Projections of token vectors to q, k and v."""

    def __init__(self, width: int, heads: int, kv_heads: int, dim: int, device, seed: int = 0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.weight = (torch.randn(width, (heads + 2 * kv_heads) * dim, generator=g, device=device) / width ** 0.5).half()

    def qkv(self, x: torch.Tensor):
        y = (x @ self.weight).view(x.shape[0], self.heads + 2 * self.kv_heads, self.dim)
        return y.split([self.heads, self.kv_heads, self.kv_heads], dim=1)


def offsets(counts, device) -> torch.Tensor:
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=device)


def run(requests: int = 4, steps: int = 6, nodes: int = 13, heads: int = 8, kv_heads: int = 2, dim: int = 64,
        width: int = 256, page: int = 16, layout: str = "bnhd", device="cuda") -> float:
    """Returns the largest difference between tree decoding and decoding token by token."""
    layer = Layer(width, heads, kv_heads, dim, device)
    prompts = [17 + 29 * b for b in range(requests)]
    longest = max(prompts) + steps * nodes
    blocks = -(-longest // page) + 1
    table = rotary_table(longest + 1, dim, device=device)
    g = torch.Generator(device=device).manual_seed(1)

    def cache():
        return PagedCache(requests, requests * blocks, page, kv_heads, dim, blocks, layout=layout, device=device)

    # ---- with trees ----
    tree = cache()
    x = torch.randn(sum(prompts), width, generator=g, device=device).half()
    step = tree.plan(offsets(prompts, device), sum(prompts))
    tree.attend(0, *layer.qkv(x), table, step)
    tree.commit(step, torch.tensor(prompts, device=device))
    kept_x, kept_out = [], []
    cu = offsets([nodes] * requests, device)
    draft = torch.Generator().manual_seed(2)
    for _ in range(steps):
        # a tree as a draft model would give it: node i hangs below one of those before it
        parents = [[-1 if i == 0 else int(torch.randint(-1, i, (1,), generator=draft)) for i in range(nodes)]
                   for _ in range(requests)]
        x_step = torch.randn(requests * nodes, width, generator=g, device=device).half()
        step = tree.plan(cu, requests * nodes,
                         parents=torch.tensor(sum(parents, []), dtype=torch.int32, device=device),
                         mask_words=-(-nodes // 32))
        out = tree.attend(0, *layer.qkv(x_step), table, step)
        # the verified path: here the last node's, in earnest what the sampled tokens say
        paths = []
        for p in parents:
            node, path = nodes - 1, []
            while node >= 0:
                path.insert(0, node)
                node = p[node]
            paths.append(path)
        kept = torch.tensor([len(p) for p in paths], device=device)
        most = max(map(len, paths))
        tree.commit(step, kept, torch.tensor([p + [0] * (most - len(p)) for p in paths], device=device))
        kept_x.append([x_step[b * nodes:(b + 1) * nodes][p] for b, p in enumerate(paths)])
        kept_out.append([out[b * nodes:(b + 1) * nodes][p] for b, p in enumerate(paths)])

    # ---- the same tokens one by one ----
    plain = cache()
    step = plain.plan(offsets(prompts, device), sum(prompts))
    plain.attend(0, *layer.qkv(x), table, step)
    plain.commit(step, torch.tensor(prompts, device=device))
    tokens = [torch.cat([s[b] for s in kept_x]) for b in range(requests)]
    outs = [[] for _ in range(requests)]
    for n in range(max(map(len, tokens))):
        live = [n < len(t) for t in tokens]
        counts = [int(alive) for alive in live]
        step = plain.plan(offsets(counts, device), sum(counts))
        x_one = torch.stack([t[n] for t, alive in zip(tokens, live) if alive])
        out = plain.attend(0, *layer.qkv(x_one), table, step)
        plain.commit(step, torch.tensor(counts, device=device))
        for row, b in enumerate(b for b in range(requests) if live[b]):
            outs[b].append(out[row])
    assert torch.equal(plain.context_lens, tree.context_lens)
    far = 0.0
    for b in range(requests):
        want = torch.stack(outs[b]).float()
        got = torch.cat([s[b] for s in kept_out]).float()
        far = max(far, float((got - want).abs().max()))
    for b in range(requests):
        tree.release(b)
    assert int(tree.num_free) == requests * blocks
    assert sorted(tree.free_blocks.tolist()) == list(range(requests * blocks))
    return far


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("requests", 4), ("steps", 6), ("nodes", 13), ("heads", 8), ("kv-heads", 2), ("dim", 64)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args()
    far = run(a.requests, a.steps, a.nodes, a.heads, a.kv_heads, a.dim)
    print(f"largest difference between tree decoding and decoding token by token: {far:.2e}")
