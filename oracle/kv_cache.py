"""Plain 64-bit restatement of the 8-bit key/value cache, its attention and
eviction, and of rotary positions (include/vicinity_gpu.h), for the tests."""
from __future__ import annotations

import math

import numpy as np


def rotary_frequencies(dim, base=10000.0, scaling="none", factor=1.0, original_length=0.0, low_turns=1.0,
                       high_turns=32.0):
    f = np.array([base ** (-2.0 * i / dim) for i in range(dim // 2)])
    if scaling == "linear":
        return f / factor
    if scaling == "by_parts":
        g = np.clip((original_length * f / (2 * math.pi) - low_turns) / (high_turns - low_turns), 0.0, 1.0)
        return (1 - g) * f / factor + g * f
    return f


def rotary(x, pos, freq, interleaved=False, magnitude=1.0, transpose=False):
    """x [tokens, heads, d] in float64."""
    r, out = 2 * len(freq), np.array(x, dtype=np.float64)
    t = np.asarray(pos, dtype=np.float64)[:, None, None] * freq
    c, s = magnitude * np.cos(t), magnitude * np.sin(t) * (-1 if transpose else 1)
    ia, ib = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = out[..., ia].copy(), out[..., ib].copy()
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    return out


def block_scale(x):
    """Smallest power of two in [2^-100, 2^120] with 127 s >= |x|; NaN for values that are not finite."""
    top = float(np.abs(x).max(initial=0.0)) if np.isfinite(x).all() else math.nan
    if math.isnan(top):
        return math.nan
    if top == 0:
        return 2.0 ** -100
    m, e = math.frexp(top)  # top = m 2^e, m in [0.5, 1)
    return 2.0 ** min(max(e - 7 + (m > 127 / 128), -100), 120)


class Head:
    """One head's keys (or values) of one sequence."""

    def __init__(self, dim, block):
        self.block, self.codes, self.scales = block, np.zeros((0, dim)), np.zeros(0)

    def __len__(self):
        return self.codes.shape[0]

    def truncate(self, n):
        self.codes, self.scales = self.codes[:n], self.scales[:-(-n // self.block)]

    def append(self, x):
        x, n, B = np.asarray(x, np.float64), len(self), self.block
        while x.shape[0]:
            room = B - n % B
            part, x = x[:room], x[room:]
            s = block_scale(part)
            if n % B:
                was = self.scales[-1]
                s = math.nan if math.isnan(s) or math.isnan(was) else max(s, was)
                if s > was:
                    self.codes[n // B * B:] = np.round(self.codes[n // B * B:] * (was / s))
                self.scales[-1] = s
            else:
                self.scales = np.append(self.scales, s)
            code = np.zeros(part.shape) if math.isnan(s) else np.clip(np.round(part / s), -127, 127)
            self.codes = np.concatenate([self.codes, code])
            n += part.shape[0]

    def values(self):
        return self.codes * np.repeat(self.scales, self.block)[:len(self), None]

    def kept(self, at):
        out, was = Head(self.codes.shape[1], self.block), self.scales[np.asarray(at, int) // self.block]
        out.codes, parts = self.codes[at].copy(), []
        for b in range(0, len(at), self.block):
            s = was[b:b + self.block].max()  # NaN if one is
            parts.append(s)
            if not math.isnan(s):
                rows = slice(b, b + self.block)
                out.codes[rows] = np.round(out.codes[rows] * (was[rows] / s)[:, None])
        out.scales = np.array(parts)
        return out


def attention(q, k, v, n_queries, scale, causal=True):
    """q [n, g, d] of one key/value head over k, v [len, d]: (out, lse,
    weights, bound terms sum p |v| and max scale sum |q k|)."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n, L = q.shape[0], k.shape[0]
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        s = scale * np.einsum("ngd,ld->ngl", q, k)
        seen = np.ones((n, 1, L), bool)
        if causal:
            seen = (np.arange(L)[None, :] < (L - n_queries + 1 + np.arange(n))[:, None])[:, None, :]
            s = np.where(seen, s, -np.inf)
        if L == 0:
            return np.zeros(q.shape), np.full(q.shape[:2], -np.inf), np.zeros(0), np.zeros(q.shape), np.zeros(q.shape[:2])
        m = s.max(-1, keepdims=True)
        m = np.where(m == -np.inf, 0.0, m)
        p = np.where(seen, np.exp(s - m), 0.0)
        l = p.sum(-1, keepdims=True)
        p = np.where(l == 0, 0.0, p / np.where(l == 0, 1.0, l))
        lse = (m + np.log(l))[..., 0]
        pv = np.where(seen[..., None], p[..., None] * v, 0.0)  # a masked NaN value is not read
        size = np.abs(scale) * np.einsum("ngd,ld->ngl", np.abs(q), np.abs(k))
    return (pv.sum(2), lse, p.sum((0, 1)), np.abs(pv).sum(2),
            np.where(seen, size, 0.0).max(-1))


def keep(weights, length, budget, recent):
    """The tokens an eviction keeps: recent ones, then by weight, ties to the older."""
    if length <= budget:
        return np.arange(length)
    old = max(0, length - recent)
    best = np.argsort(-np.asarray(weights[:old], np.float64), kind="stable")[:budget - (length - old)]
    return np.sort(np.concatenate([best, np.arange(old, length)]))
