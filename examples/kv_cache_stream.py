"""Streaming decode with a bounded key/value cache.

One attention layer of a batch of sequences, fed with random projections in
place of a model's: a prompt goes through rotary positions, the 8-bit cache and
chunked attention that accumulates each cached token's weight; then every step
adds one token per sequence, and whenever the sequences have grown by `grow`
tokens they are cut back to `budget` by accumulated weight.  Each sequence owns
two slots of the cache and moves to its other one with every eviction.

    python examples/kv_cache_stream.py [--steps 200]

prints the time of a step, and how close the outputs are to attention in full
precision over all tokens (the keys have a few directions that queries look
for, so most of the attention survives the evictions).
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from vicinity_b200 import KVCache, Rotary  # noqa: E402


class StreamingAttention:
    def __init__(self, seqs: int, heads: int, kv_heads: int, dim: int, budget: int, recent: int, grow: int,
                 chunk: int):
        self.seqs, self.heads, self.kv_heads, self.dim = seqs, heads, kv_heads, dim
        self.budget, self.recent, self.limit = budget, recent, budget + grow
        self.rotary = Rotary(dim)
        self.cache = KVCache(2 * seqs, self.limit + chunk, kv_heads, dim)
        self.slot = list(range(seqs))           # where each sequence lives: its slot or the one seqs further
        self.position = [0] * seqs

    def _counts(self, n: int) -> list[int]:
        counts = [0] * (2 * self.seqs)
        for s in self.slot:
            counts[s] = n
        return counts

    def step(self, q, k, v):
        """Attention outputs of n new tokens per sequence: q [seqs, n, heads,
        dim], k and v [seqs, n, kv_heads, dim] before rotary positions."""
        n = q.shape[1]
        # the packed tensors are in the order of the cache's slots
        order = sorted(range(self.seqs), key=lambda s: self.slot[s])
        flat = [x[order].reshape(self.seqs * n, -1, self.dim) for x in (q, k, v)]
        at = torch.tensor([self.position[s] for s in order], device=q.device)
        positions = (at[:, None] + torch.arange(n, device=q.device)).reshape(-1)
        self.rotary.apply(positions, flat[0], flat[1])
        counts = self._counts(n)
        self.cache.append(flat[1], flat[2], counts)
        out = torch.empty_like(flat[0])
        self.cache.attend(flat[0], counts, out, accumulate=True)
        self.position = [p + n for p in self.position]
        lengths = self.cache.lengths
        full = [s for s in range(self.seqs) if lengths[self.slot[s]] > self.limit]
        if full:
            src = [self.slot[s] for s in full]
            dst = [(x + self.seqs) % (2 * self.seqs) for x in src]
            self.cache.evict(src, dst, self.budget, self.recent)
            keep = self.cache.lengths
            keep[src] = 0
            self.cache.truncate(keep)
            for s, d in zip(full, dst):
                self.slot[s] = d
        back = torch.empty(self.seqs, dtype=torch.long, device=q.device)
        back[torch.tensor(order, device=q.device)] = torch.arange(self.seqs, device=q.device)
        return out.view(self.seqs, n, self.heads, self.dim)[back]


def projections(g, seqs, n, heads, kv_heads, dim):
    """Random queries, keys and values; one key in 16 lies along a direction
    that the queries of its head look for."""
    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    q, k, v = normal(seqs, n, heads, dim), normal(seqs, n, kv_heads, dim), normal(seqs, n, kv_heads, dim)
    # the second half of the dimensions turns so slowly that it hardly depends on the position
    q[..., dim // 2 - 8:dim // 2] += 2.0
    k[:, ::16, :, dim // 2 - 8:dim // 2] += 3.0
    return [x.to(torch.bfloat16) for x in (q, k, v)]


def full_attention(rotary, q, k, v, keys, values, start):
    """The same step without a bound and in f32; keys and values grow."""
    n, group = q.shape[1], q.shape[2] // k.shape[2]
    positions = torch.arange(start, start + n, device="cuda").repeat(q.shape[0])
    q, k = q.float().flatten(0, 1), k.float().flatten(0, 1)
    rotary.apply(positions, q, k)
    q, k = q.unflatten(0, (-1, n)), k.unflatten(0, (-1, n))
    keys.append(k)
    values.append(v.float())
    kk, vv = (torch.cat(x, 1).repeat_interleave(group, 2) for x in (keys, values))
    s = torch.einsum("snhd,slhd->shnl", q, kk) * q.shape[-1] ** -0.5
    hidden = torch.arange(kk.shape[1], device="cuda") > start + torch.arange(n, device="cuda")[:, None]
    return torch.einsum("shnl,slhd->snhd", torch.softmax(s.masked_fill(hidden, -torch.inf), -1), vv)


def main(argv=None) -> float:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=1500)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--budget", type=int, default=512)
    a = ap.parse_args(argv)
    heads, kv_heads, dim, chunk = 16, 4, 128, 500
    g = torch.Generator(device="cuda").manual_seed(0)
    layer = StreamingAttention(a.seqs, heads, kv_heads, dim, a.budget, recent=64, grow=64, chunk=chunk)
    keys, values, start, near = [], [], 0, []
    sizes = [min(chunk, a.prompt - x) for x in range(0, a.prompt, chunk)] + [1] * a.steps
    spent = []
    for n in sizes:
        q, k, v = projections(g, a.seqs, n, heads, kv_heads, dim)
        before, after = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        before.record()
        out = layer.step(q, k, v)
        after.record()
        want = full_attention(layer.rotary, q, k, v, keys, values, start)
        start += n
        near.append(torch.nn.functional.cosine_similarity(out.float(), want, dim=-1).mean())
        spent.append((n, before, after))
    torch.cuda.synchronize()
    one = sorted(b.elapsed_time(c) for n, b, c in spent if n == 1)
    near = torch.stack(near).cpu()
    first = len(sizes) - a.steps
    print(f"{a.seqs} sequences, {start} tokens each, {int(layer.cache.lengths.max())} kept; "
          f"cosine to full attention: prompt {near[:first].mean():.4f}, steps {near[first:].mean():.4f}")
    if one:
        print(f"a step: {1e3 * one[len(one) // 2]:.0f} us (median of {len(one)}, evictions among them)")
    return float(near.mean())


if __name__ == "__main__":
    main()
