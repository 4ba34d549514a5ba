"""Next-item decoding with a paged, budgeted key-value cache.

A small sequence model over the lookup layers: item embeddings from a table in
HBM (NVEmbedding, GPULayer), a few attention blocks whose keys and values live
in KVCache pages, and one new item per user and step, the best one or one drawn
from the likely ones.  Every user's cache holds at most about `budget` items: once
it is a page over, the items that have received the least attention are evicted,
except the first few and the latest.

  python examples/sequence_decode.py --users 16 --steps 64
  python examples/sequence_decode.py --users 16 --steps 64 --mxfp4 --norms --temperature 0.8 --top-p 0.9
"""
import argparse
import os
import sys
import time

import torch
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "nv-embedding-cache_amd")
if PKG not in sys.path:
    sys.path.insert(0, PKG)

from pynve.torch.nve_kv import KVCache  # noqa: E402
from pynve.torch.nve_layers import LayerType, NVEmbedding  # noqa: E402
from pynve.torch.nve_sample import sample_tokens  # noqa: E402


class SequenceDecoder:
    """`users` sequences decoded together; `layers` attention blocks of `q_heads` query and
    `kv_heads` key heads over item rows of `width` values."""

    def __init__(self, items, users, width=256, layers=2, q_heads=8, kv_heads=2, budget=256, sinks=4, recent=32,
                 page=16, longest=4096, dtype=torch.float16, cache_dtype=None, norms=False, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        dim = width // q_heads
        draw = lambda *s: (torch.randn(s, device="cuda", generator=g) * s[0] ** -0.5).to(dtype)  # noqa: E731
        self.emb = NVEmbedding(items, width, dtype, LayerType.GPULayer, optimize_for_training=False)
        self.emb.weight.data.copy_(torch.randn((items, width), device="cuda", generator=g))
        self.blocks = [{"qkv": draw(width, (q_heads + 2 * kv_heads) * dim), "out": draw(q_heads * dim, width),
                        "up": draw(width, 2 * width), "down": draw(2 * width, width),
                        # the weights of the query and key heads' norms
                        **({n: torch.ones(dim, device="cuda", dtype=dtype) for n in ("q_norm", "k_norm")} if norms else {})}
                       for _ in range(layers)]
        self.q_heads, self.kv_heads, self.dim, self.dtype = q_heads, kv_heads, dim, dtype
        self.budget, self.sinks, self.recent, self.page = budget, sinks, recent, page
        # a sequence grows to a page over the budget before it is cut
        self.pages_each = -(-(budget + page) // page)
        self.caches = [KVCache(users * self.pages_each, kv_heads, dim, page=page, dtype=cache_dtype or dtype)
                       for _ in range(layers)]
        # all sequences of all layers have the same lengths, so one table of pages serves every cache
        self.tables = torch.arange(users * self.pages_each, device="cuda", dtype=torch.int32).view(users, -1)
        self.lengths = torch.zeros(users, device="cuda", dtype=torch.int32)
        self.length = self.seen = 0
        self.users = torch.arange(users, device="cuda")
        angle = torch.arange(longest, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, dim, 2, device="cuda") / dim)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()

    @torch.no_grad()
    def step(self, items):
        """The hidden rows after one more item per user (int64 [users])."""
        x = self.emb(items)
        slots = self.caches[0].slots(self.tables, self.users, torch.full_like(self.users, self.length))
        at = torch.full_like(self.lengths, self.seen)
        self.lengths += 1
        for w, cache in zip(self.blocks, self.caches):
            qkv = F.layer_norm(x, x.shape[1:]) @ w["qkv"]
            q, k, v = qkv.view(len(items), -1, self.dim).split([self.q_heads, self.kv_heads, self.kv_heads], 1)
            q = cache.append(k, v, slots, q=q, positions=at, cos_sin=self.cos_sin, q_norm=w.get("q_norm"),
                             k_norm=w.get("k_norm"))
            x = x + cache.attend(q, self.tables, self.lengths).flatten(1) @ w["out"]
            x = x + F.gelu(F.layer_norm(x, x.shape[1:]) @ w["up"]) @ w["down"]
        self.length += 1
        self.seen += 1
        if self.length == self.budget + self.page:
            for cache in self.caches:
                new = cache.evict(self.tables, self.lengths, self.budget, sinks=self.sinks, recent=self.recent)
            self.lengths.copy_(new)
            self.length = self.budget
        return x

    @torch.no_grad()
    def next_items(self, hidden, candidates, u=None, **limits):
        """The best of `candidates` (int64) for every user, or, with random numbers `u` (float32 [users]), one drawn
        within sample_tokens' limits."""
        scores = hidden @ self.emb(candidates).t()
        return candidates[scores.argmax(1) if u is None else sample_tokens(scores, u, **limits)]


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--items", type=int, default=100000)
    ap.add_argument("--users", type=int, default=16)
    ap.add_argument("--steps", type=int, default=400)
    ap.add_argument("--budget", type=int, default=256)
    ap.add_argument("--e4m3", action="store_true", help="keep keys and values in 8 bits")
    ap.add_argument("--mxfp4", action="store_true", help="keep keys and values in 4 bits")
    ap.add_argument("--norms", action="store_true", help="norm the query and key heads")
    ap.add_argument("--temperature", type=float, default=0.0, help="draw items; 0 takes the best")
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--min-p", type=float, default=0.0)
    a = ap.parse_args(argv)
    model = SequenceDecoder(a.items, a.users, budget=a.budget, longest=a.steps + 1, norms=a.norms,
                            cache_dtype=torch.float4_e2m1fn_x2 if a.mxfp4 else torch.float8_e4m3fn if a.e4m3 else None)
    limits = {"temperature": a.temperature, "top_k": a.top_k, "top_p": a.top_p, "min_p": a.min_p}
    candidates = torch.arange(0, a.items, max(1, a.items // 1000), device="cuda")
    items = torch.randint(0, a.items, (a.users,), device="cuda")
    model.step(items)
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(a.steps - 1):
        u = torch.rand(a.users, device="cuda") if a.temperature > 0 else None
        items = model.next_items(model.step(items), candidates, u, **(limits if u is not None else {}))
    torch.cuda.synchronize()
    spent = (time.perf_counter() - start) / max(1, a.steps - 1)
    print(f"{a.users} users, {a.steps} steps: {spent * 1e6:.0f} us a step, {model.length} of {model.seen} items kept, "
          f"last items {items[:4].tolist()}")
    return items


if __name__ == "__main__":
    main()
