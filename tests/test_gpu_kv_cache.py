"""Rotary positions and the 8-bit key/value cache on the GPU against the plain
64-bit restatement in oracle/kv_cache.py.

Stored codes, scales and evictions are exact (power-of-two scales), so they
are compared bit for bit.  Bounds of the rest, with u = 2^-24 and u_out the
output type's unit roundoff:
  rotary     |err| <= u_out |out| + 8 u m (|a| + |b|): angle rounded to f32 as a
             fraction of a turn, sine and cosine to 2 ulp, three roundings
  scores     |err| <= e = (d + 16) u S, S = scale sum |q_i k_i|: f32 sums of exact
             products in any order, one rounding of the factor
  lse        |err| <= e + 16 u (1 + |lse|)
  weights    |err| <= (2 e + 32 u (1 + |lse|)) w
  out        |err| <= 1.01 u_out |out| + (2^-11 + 2 e + 32 u (1 + |lse|)) sum p |v| + n 2^-36 max |v|:
             probabilities rounded to binary16 (2^-12, doubled), those of n tokens
             below its range, 2^-38 of the largest, to 0
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from oracle import kv_cache as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
ROUND = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # bf16: 8 significant bits


def _types():
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _rand(g, *shape, dtype="f32", scale=1.0):
    x = torch.from_numpy((g.standard_normal(shape) * scale).astype(np.float32)).to(_types()[dtype])
    return x.cuda()


def _np(x):
    return x.detach().double().cpu().numpy()


# ---- rotary -----------------------------------------------------------------


def _rotary_bound(x, want, freq, interleaved, m, dtype):
    r = 2 * len(freq)
    size, pairs = np.zeros_like(want), np.abs(_np(x))
    ia, ib = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    size[..., ia] = size[..., ib] = pairs[..., ia] + pairs[..., ib]
    tiny = 2.0 ** -25 if dtype == "f16" else 0.0  # half the smallest binary16
    return 1.01 * ROUND[dtype] * np.abs(want) + 8 * U * m * size + tiny


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,hq,hk,d,rot", [(1, 1, 1, 32, 32), (5, 8, 2, 128, 128), (33, 3, 1, 96, 64),
                                                (700, 12, 4, 64, 64), (7, 2, 2, 100, 50), (9, 1, 3, 10, 2),
                                                (3, 2, 1, 256, 256)])
def test_rotary(tokens, hq, hk, d, rot, layout, dtype):
    from vicinity_b200 import Rotary

    g = np.random.default_rng(tokens + d)
    pos = g.integers(0, 1 << 20, tokens)
    pos[0] = 0
    pos[-1] = (1 << 31) + 5 if tokens > 1 else 0
    q, k = _rand(g, tokens, hq, d, dtype=dtype), _rand(g, tokens, hk, d, dtype=dtype)
    scaled = dict(scaling="by_parts", factor=8.0, original_length=4096.0, magnitude=1.25)
    r = Rotary(rot, base=500.0, layout=layout, **scaled)
    freq = ref.rotary_frequencies(rot, 500.0, "by_parts", 8.0, 4096.0)
    assert np.allclose(r.frequencies(), freq, rtol=1e-14)
    p = torch.from_numpy(pos).cuda()
    for transpose in (False, True):
        oq, ok = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
        r.apply(p, q, k, out_q=oq, out_k=ok, transpose=transpose)
        for x, got in ((q, oq), (k, ok)):
            want = ref.rotary(_np(x), pos, r.frequencies(), layout == "interleaved", 1.25, transpose)
            err = np.abs(_np(got) - want)
            assert (err <= _rotary_bound(x, want, freq, layout == "interleaved", 1.25, dtype)).all(), err.max()
        # in place, and one tensor alone
        qi = q.clone()
        r.apply(p, qi, transpose=transpose)
        assert torch.equal(qi, oq)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_strides_and_alignment(layout):
    # head-major storage, an odd first element, a broadcast input: the same as contiguous copies
    from vicinity_b200 import Rotary

    g = np.random.default_rng(3)
    t, h, d = 19, 4, 64
    r = Rotary(d, layout=layout, scaling="linear", factor=2.0)
    pos = torch.arange(100, 100 + t).cuda()
    base = _rand(g, h, t, d, dtype="bf16").transpose(0, 1)
    flat = _rand(g, t * h * d + 1, dtype="bf16")
    odd = flat[1:].view(t, h, d)
    wide = _rand(g, t, 1, d, dtype="bf16").expand(t, h, d)
    for x in (base, odd, wide):
        want, got = torch.empty(t, h, d, dtype=x.dtype, device="cuda"), torch.empty(h, t, d, dtype=x.dtype, device="cuda")
        r.apply(pos, x.contiguous(), out_q=want)
        r.apply(pos, x, out_q=got.transpose(0, 1))
        assert torch.equal(got.transpose(0, 1), want)


def test_rotary_gradient():
    # the transposed map against differences of the map in 64 bits, and as the
    # adjoint: <R x, y> = <x, R^T y>
    from vicinity_b200 import Rotary

    g = np.random.default_rng(8)
    t, h, d, rot = 6, 2, 24, 16
    r = Rotary(rot, layout="interleaved", magnitude=0.75)
    pos = np.array([0, 1, 17, 300, 4000, 70000])
    x, y = g.standard_normal((t, h, d)), g.standard_normal((t, h, d)).astype(np.float32)
    dx = torch.empty(t, h, d, device="cuda")
    r.apply(torch.from_numpy(pos).cuda(), torch.from_numpy(y).cuda(), out_q=dx, transpose=True)
    freq, eps = r.frequencies(), 1e-3
    for i in ((0, 0, 3), (2, 1, 0), (3, 1, 15), (5, 0, 8), (4, 1, 20)):
        up, down = x.copy(), x.copy()
        up[i] += eps
        down[i] -= eps
        f = [(ref.rotary(z, pos, freq, True, 0.75) * y).sum() for z in (up, down)]
        # linear map: the difference quotient is exact up to rounding (~1e-11)
        assert abs((f[0] - f[1]) / (2 * eps) - float(dx[i])) <= 1e-9 + 8 * U * 0.75 * 2 * np.abs(y).max()


def test_rotary_in_a_captured_graph_and_on_a_stream():
    from vicinity_b200 import Rotary

    g = np.random.default_rng(4)
    q = _rand(g, 8, 2, 32, dtype="f16")
    pos, out, want = torch.arange(8).cuda(), torch.empty_like(q), torch.empty_like(q)
    r = Rotary(32)
    r.apply(pos, q, out_q=want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        r.apply(pos, q, out_q=out, stream=torch.cuda.current_stream().cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ---- cache ------------------------------------------------------------------


class Mirror:
    """A KVCache and its restatement, driven together."""

    def __init__(self, seqs, capacity, heads, d, block):
        from vicinity_b200 import KVCache

        self.cache = KVCache(seqs, capacity, heads, d, block_tokens=block)
        self.heads, self.d, self.block, self.seqs = heads, d, block, seqs
        self.k = [[ref.Head(d, block) for _ in range(heads)] for _ in range(seqs)]
        self.v = [[ref.Head(d, block) for _ in range(heads)] for _ in range(seqs)]
        self.w = [[np.zeros(0) for _ in range(heads)] for _ in range(seqs)]

    def append(self, counts, k, v, stream=None):
        self.cache.append(k, v, counts, stream=stream)
        kn, vn, row = _np(k), _np(v), 0
        for s, c in enumerate(counts):
            for h in range(self.heads):
                self.k[s][h].append(kn[row:row + c, h])
                self.v[s][h].append(vn[row:row + c, h])
                self.w[s][h] = np.concatenate([self.w[s][h], np.zeros(c)])
            row += c

    def fill(self, g, counts, dtype="bf16", scale=1.0):
        n = sum(counts)
        self.append(counts, _rand(g, n, self.heads, self.d, dtype=dtype, scale=scale),
                    _rand(g, n, self.heads, self.d, dtype=dtype, scale=scale))

    def truncate(self, lengths):
        self.cache.truncate(lengths)
        for s, n in enumerate(lengths):
            for h in range(self.heads):
                self.k[s][h].truncate(n)
                self.v[s][h].truncate(n)
                self.w[s][h] = self.w[s][h][:n]

    def check(self):
        torch.cuda.synchronize()
        assert self.cache.lengths.tolist() == [len(h[0]) for h in self.k]
        for s in range(self.seqs):
            kc, ks, vc, vs, _ = self.cache.export(s)
            for h in range(self.heads):
                for codes, scales, want in ((kc, ks, self.k[s][h]), (vc, vs, self.v[s][h])):
                    assert np.array_equal(scales[h], want.scales, equal_nan=True), (s, h)
                    sound = ~np.isnan(np.repeat(want.scales, self.block)[:len(want)])
                    assert np.array_equal(codes[h][sound], want.codes[sound]), (s, h)

    def attend(self, counts, q, dtype, scale=None, causal=True, accumulate=False, out=None, stream=None):
        n, hq = q.shape[0], q.shape[1]
        g = hq // self.heads
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda") if out is None else out
        lse = torch.full((n, hq), 7.0, device="cuda")
        self.cache.attend(q, counts, out, lse=lse, scale=scale, causal=causal, accumulate=accumulate, stream=stream)
        torch.cuda.synchronize()
        scale = self.d ** -0.5 if scale is None else scale
        qn, on, ln, row = _np(q), _np(out), _np(lse), 0
        weights = torch.as_tensor(self.cache.weights, device="cuda").double().cpu().numpy()
        for s, c in enumerate(counts):
            for h in range(self.heads if c else 0):
                heads = slice(h * g, (h + 1) * g)
                o, want_lse, w, size, top = ref.attention(qn[row:row + c, heads], self.k[s][h].values(),
                                                          self.v[s][h].values(), c, scale, causal)
                e = (self.d + 16) * U * top
                soft = np.where(np.isfinite(want_lse), np.abs(want_lse), 0.0)
                got, got_lse = on[row:row + c, heads], ln[row:row + c, heads]
                fine = np.isfinite(want_lse)
                assert np.array_equal(np.isnan(want_lse), np.isnan(got_lse))
                assert np.array_equal(want_lse == -np.inf, got_lse == -np.inf)
                err = np.abs(got_lse[fine] - want_lse[fine])
                assert (err <= (e + 16 * U * (1 + soft))[fine]).all(), (s, h, err.max())
                tol = 1.01 * ROUND[dtype] * np.abs(o) + (2.0 ** -11 + 2 * e + 32 * U * (1 + soft))[..., None] * size
                tol += 2.0 ** -24 if dtype == "f16" else 0.0
                tol += len(self.v[s][h]) * 2.0 ** -36 * np.nan_to_num(np.abs(self.v[s][h].values())).max(initial=0.0)
                assert np.array_equal(np.isnan(o), np.isnan(got)), (s, h)
                ok = ~np.isnan(o)
                assert (np.abs(got - o)[ok] <= tol[ok]).all(), (s, h, np.nanmax(np.abs(got - o) / (tol + 1e-300)))
                assert (got[want_lse == -np.inf] == 0).all()
                if accumulate:
                    rel = (2 * e + 32 * U * (1 + soft))[fine].max(initial=0.0)
                    old, now = self.w[s][h], weights[s, h, :len(self.w[s][h])]
                    assert np.array_equal(np.isnan(old + w), np.isnan(now)), (s, h)
                    err = np.nan_to_num(np.abs(now - (old + w)))
                    assert (err <= np.nan_to_num(rel * w + 4 * U * (old + w)) + 1e-12).all(), (s, h, err.max())
                    # later steps and evictions start from what the cache holds
                    self.w[s][h] = now.copy()
            row += c
        return out


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_append_and_read(block, d, dtype):
    g = np.random.default_rng(block + d)
    m = Mirror(4, 333, 3, d, block)
    for step, counts in enumerate([[1, 0, 17, 200], [1, 0, block - 1, 1], [block, 0, 1, 3], [0, 0, 0, 0], [40, 0, 2, 129]]):
        # growing magnitudes make the scales of blocks with tokens grow
        m.fill(g, counts, dtype, scale=2.0 ** (step % 3) * 0.7)
    m.check()
    starts, counts = [0, 0, 5, 100], [43, 0, 1, 233]
    n = sum(counts)
    k, v = (torch.full((n, 3, d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    m.cache.read(starts, counts, k, v)
    row = 0
    for s, c in enumerate(counts):
        for h in range(3):
            assert np.array_equal(_np(k)[row:row + c, h], m.k[s][h].values()[starts[s]:starts[s] + c])
            assert np.array_equal(_np(v)[row:row + c, h], m.v[s][h].values()[starts[s]:starts[s] + c])
        row += c


def test_append_edges_of_the_scales():
    # zeros, the powers of two where the scale steps, subnormals, the largest
    # floats, infinities and NaN, each in a block of its own
    rows = [[0.0], [127.0], [127.0 * (1 + 2.0 ** -20)], [128.0], [2.0 ** -140], [3.0e38, -3.4e38], [math.inf], [math.nan],
            [1.0, -1.0], [0.5, 1.5, 2.5, 127.0, -0.5, -1.5, -2.5]]
    x = np.zeros((16 * len(rows), 1, 32), np.float32)
    for i, r in enumerate(rows):
        x[16 * i, 0, :len(r)] = r
    m = Mirror(1, 16 * len(rows) + 16, 1, 32, 16)
    t = torch.from_numpy(x).cuda()
    m.append([x.shape[0]], t, t.clone())
    m.check()
    # a block that was given NaN stays NaN until it starts afresh
    m.append([1], torch.full((1, 1, 32), math.nan, device="cuda"), torch.ones(1, 1, 32, device="cuda"))
    m.append([1], torch.ones(1, 1, 32, device="cuda"), torch.ones(1, 1, 32, device="cuda"))
    m.check()
    m.truncate([x.shape[0]])
    m.append([3], torch.ones(3, 1, 32, device="cuda"), torch.ones(3, 1, 32, device="cuda"))
    m.check()


def test_append_strided_broadcast_and_unaligned():
    g = np.random.default_rng(5)
    for dtype in ("f32", "bf16"):
        m = Mirror(2, 100, 4, 64, 32)
        k = _rand(g, 4, 70, 64, dtype=dtype).transpose(0, 1)           # head-major
        v = _rand(g, 70, 1, 64, dtype=dtype).expand(70, 4, 64)         # one head for all
        m.append([30, 40], k, v)
        flat = _rand(g, 20 * 4 * 65 + 1, dtype=dtype)
        odd = flat[1:].view(20, 4, 65)[..., :64]                       # rows that start anywhere
        m.append([20, 0], odd, odd)
        m.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,block,heads,group", [(32, 16, 1, 1), (64, 32, 2, 4), (96, 64, 3, 7), (128, 128, 2, 8),
                                                 (128, 64, 1, 33), (64, 16, 5, 2)])
def test_attend_single_tokens(d, block, heads, group, dtype):
    g = np.random.default_rng(d + group)
    m = Mirror(6, 700, heads, d, block)
    m.fill(g, [1, 0, 15, 129, 700, 300], scale=1.5)
    q = _rand(g, 6, heads * group, d, dtype=dtype, scale=2.0)
    m.attend([1] * 6, q, dtype, accumulate=True)
    m.attend([1] * 6, q, dtype, accumulate=True, scale=0.03)  # weights add up
    m.attend([0, 0, 1, 0, 1, 0], q[:2], dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,block,heads,group,counts", [
    (64, 32, 2, 2, [3, 2, 0, 5]), (128, 64, 1, 4, [40, 1, 33, 0]), (96, 16, 2, 3, [129, 0, 64, 7]),
    (32, 128, 1, 8, [17, 16, 15, 1]), (128, 32, 2, 1, [257, 3, 0, 130])])
@pytest.mark.parametrize("causal", [True, False])
def test_attend_several_tokens(d, block, heads, group, counts, causal, dtype):
    g = np.random.default_rng(d + group + sum(counts))
    m = Mirror(4, 640, heads, d, block)
    m.fill(g, [300, 2, 64, 0])        # the last sequence is empty but for its own queries
    m.fill(g, counts)
    q = _rand(g, sum(counts), heads * group, d, dtype=dtype, scale=2.0)
    m.attend(counts, q, dtype, causal=causal, accumulate=True)


def test_attend_rows_that_see_nothing():
    # more queries than tokens: the first ones see none; an empty sequence
    g = np.random.default_rng(2)
    for counts in ([20, 3, 1], [150, 1, 140], [1, 300, 1]):
        m = Mirror(3, 256, 2, 64, 16)
        m.fill(g, [7, 0, 130])
        q = _rand(g, sum(counts), 4, 64, dtype="bf16")
        m.attend(counts, q, "bf16", accumulate=True)
        m.attend(counts, q, "bf16", causal=False)


def test_attend_does_not_see_what_is_masked():
    # blocks that read as NaN, and stale tokens past a truncation, reach no
    # query that does not see them
    g = np.random.default_rng(6)
    for counts in ([2, 1], [40, 33]):
        m = Mirror(2, 256, 1, 64, 16)
        m.fill(g, [100, 96])
        bad = torch.full((60, 1, 64), math.nan, device="cuda")
        m.append([30, 30], bad, bad)     # the first sequence's last block has 4 older tokens: they read as NaN
        m.truncate([100, 96])
        q = _rand(g, sum(counts), 2, 64, dtype="bf16")
        m.attend(counts, q, "bf16", accumulate=True)
        # ... and every query that sees them is NaN
        m.append([0, 16], bad[:16], bad[:16])
        m.attend([0, counts[1]], q[:counts[1]], "bf16")


def test_attend_scores_far_apart():
    # huge scores (one token takes all), equal scores, negative and zero scale
    g = np.random.default_rng(7)
    for n in (1, 48):
        m = Mirror(1, 400, 2, 128, 64)
        m.fill(g, [333], scale=8.0)
        q = _rand(g, n, 4, 128, dtype="bf16", scale=8.0)
        for scale in (1.0, -0.05, 0.0):
            m.attend([n], q, "bf16", scale=scale, accumulate=True)
        m.attend([n], q * 0, "bf16")
        # values and keys of very different magnitudes from block to block
        m.fill(g, [60], scale=2.0 ** -30)
        m.fill(g, [3], scale=2.0 ** 20)
        m.attend([n], (q.float() * 2.0 ** -24).to(q.dtype), "bf16")


def test_attend_strides_and_streams():
    g = np.random.default_rng(9)
    m = Mirror(2, 300, 2, 64, 32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    m.fill(g, [200, 131])
    for n in (1, 20):
        q = _rand(g, 4, 2 * n, 64, dtype="bf16").transpose(0, 1)
        out = torch.empty(4, 2 * n, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
        torch.cuda.synchronize()
        m.attend([n, n], q, "bf16", out=out, stream=s.cuda_stream)
        flat = _rand(g, 2 * n * 4 * 67 + 1, dtype="f16")
        odd = flat[1:].view(2 * n, 4, 67)[..., 1:65]
        m.attend([n, n], odd, "f16", accumulate=True)


def test_attend_is_the_same_in_every_run_and_ordered_across_streams():
    g = np.random.default_rng(10)
    m = Mirror(3, 4000, 2, 128, 64)
    m.fill(g, [4000, 1, 777])
    for n in (1, 100):
        q = _rand(g, 3 * n, 8, 128, dtype="bf16")
        out = [torch.empty_like(q) for _ in range(4)]
        streams = [torch.cuda.Stream() for _ in out]
        torch.cuda.synchronize()
        for o, st in zip(out, streams):
            m.cache.attend(q, [n] * 3, o, accumulate=True, stream=st.cuda_stream)
        torch.cuda.synchronize()
        for o in out[1:]:
            assert torch.equal(o, out[0])


def test_long_sequence_offsets_past_32_bits():
    # the last sequence's codes lie beyond 4 GiB: [17][2][1_100_032][128]
    from vicinity_b200 import KVCache

    cap, d = 1_100_000, 128
    cache = KVCache(17, cap, 2, d, block_tokens=64)
    g = torch.Generator(device="cuda").manual_seed(1)
    n = cap - 3
    k = torch.randn(n, 2, d, generator=g, device="cuda", dtype=torch.float32).to(torch.bfloat16)
    v = torch.randn(n, 2, d, generator=g, device="cuda", dtype=torch.float32).to(torch.bfloat16)
    counts = [0] * 16 + [n]
    cache.append(k, v, counts)
    kr, vr = torch.empty(500, 2, d, dtype=torch.bfloat16, device="cuda"), torch.empty(500, 2, d, dtype=torch.bfloat16, device="cuda")
    cache.read([0] * 16 + [n - 500], [0] * 16 + [500], kr, vr)
    tail = ref.Head(d, 64)
    first = (n - 500) // 64 * 64
    tail.append(_np(k[first:, 1]))
    assert np.array_equal(_np(kr[:, 1]), tail.values()[n - 500 - first:])
    q = torch.randn(1, 4, d, generator=g, device="cuda").to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty(1, 4, device="cuda")
    cache.attend(q, [0] * 16 + [1], out, lse=lse, accumulate=True)
    # the same attention in 64 bits on the GPU, from the values read back
    kk, vv = torch.empty(n, 2, d, dtype=torch.bfloat16, device="cuda"), torch.empty(n, 2, d, dtype=torch.bfloat16, device="cuda")
    cache.read([0] * 17, counts, kk, vv)
    for h in range(4):
        s = (kk[:, h // 2].double() @ q[0, h].double()) / math.sqrt(d)
        p = torch.softmax(s, 0)
        o = p @ vv[:, h // 2].double()
        size = p @ vv[:, h // 2].double().abs()
        assert abs(float(lse[0, h]) - float(torch.logsumexp(s, 0))) <= 1e-4
        assert ((out[0, h].double() - o).abs() <= 1.01 * 2.0 ** -8 * o.abs() + (2.0 ** -11 + 1e-4) * size).all()
    w = torch.as_tensor(cache.weights, device="cuda")
    assert abs(float(w[16].double().sum()) - 4.0) <= 1e-3 and float(w[:16].abs().sum()) == 0.0


# ---- eviction ---------------------------------------------------------------


@pytest.mark.parametrize("d,block,heads", [(32, 16, 1), (64, 64, 3), (96, 32, 2), (128, 128, 2)])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (100, 0), (100, 33), (257, 257), (900, 5)])
def test_evict(budget, recent, d, block, heads):
    g = np.random.default_rng(budget + d)
    lens = [0, 1, budget, min(budget + 1, 900), 900]
    n = len(lens)
    m = Mirror(2 * n, 900, heads, d, block)
    for part in range(3):  # blocks of different scales
        m.fill(g, [(x * (part + 1)) // 3 - (x * part) // 3 for x in lens] + [0] * n, scale=3.0 ** part)
    m.fill(g, [0] * n + [37] * n)  # what the destinations held is replaced
    weights = torch.as_tensor(m.cache.weights, device="cuda")
    w = torch.from_numpy(g.exponential(size=(n, heads, 900)).astype(np.float32))
    w[torch.from_numpy(g.random((n, heads, 900)) < 0.4)] = 0.0   # many ties
    w[:, :, ::7] = 1.5
    weights[:n] = w.cuda()
    kept = torch.full((n, heads, budget), 7, dtype=torch.int32, device="cuda")
    m.cache.evict(list(range(n)), list(range(n, 2 * n)), budget, recent, kept=kept)
    torch.cuda.synchronize()
    for s, length in enumerate(lens):
        for h in range(heads):
            at = ref.keep(w[s, h].numpy(), length, budget, recent)
            assert np.array_equal(kept[s, h].cpu().numpy(), np.pad(at, (0, budget - len(at)), constant_values=-1))
            m.k[n + s][h], m.v[n + s][h] = m.k[s][h].kept(at), m.v[s][h].kept(at)
            want = np.pad(w[s, h].numpy()[at], (0, budget - len(at)))
            assert np.array_equal(weights[n + s, h, :budget].cpu().numpy(), want)
    m.check()
    # what is left is attended to and appended to
    m.fill(g, [0] * n + [min(2, 900 - min(x, budget)) for x in lens])
    q = _rand(g, n, heads, d, dtype="bf16")
    m.attend([0] * n + [1] * n, q, "bf16")


def test_evict_long_rows_and_special_weights():
    g = np.random.default_rng(12)
    m = Mirror(2, 40_000, 2, 32, 64)
    m.fill(g, [40_000, 0])
    weights = torch.as_tensor(m.cache.weights, device="cuda")
    w = g.random((2, 40_000)).astype(np.float32)
    w[0] = 0.25                                # all equal: the oldest stay
    w[1, 1000:3000] = np.inf
    w[1, 3000] = np.nan                        # counts as the largest
    w[1, 5000:9000] = 1e-42                    # subnormals keep their order
    w[1, 9000:30_000] = -0.0                   # as 0
    weights[0, :, :40_000] = torch.from_numpy(w).cuda()
    for budget, recent in ((5_000, 100), (39_999, 0), (2_500, 2_400)):
        kept = torch.empty(1, 2, budget, dtype=torch.int32, device="cuda")
        m.cache.evict([0], [1], budget, recent, kept=kept)
        order = np.where(np.isnan(w), np.inf, w).astype(np.float64)
        order[np.isnan(w)] = 1e308
        order[np.isinf(w)] = 1e307
        for h in range(2):
            assert np.array_equal(kept[0, h].cpu().numpy(), ref.keep(order[h], 40_000, budget, recent))


def test_evict_poisoned_blocks():
    g = np.random.default_rng(13)
    m = Mirror(2, 128, 1, 32, 16)
    m.fill(g, [40, 0])
    bad = torch.full((1, 1, 32), math.inf, device="cuda")
    m.append([1, 0], bad, torch.ones_like(bad))
    m.fill(g, [40, 0])
    m.cache.evict([0], [1], 30, 10)
    at = ref.keep(np.zeros(81), 81, 30, 10)
    m.k[1][0], m.v[1][0] = m.k[0][0].kept(at), m.v[0][0].kept(at)
    m.check()


# ---- whole sequences ---------------------------------------------------------


def test_load_and_export_round_trip():
    from vicinity_b200 import KVCache

    g = np.random.default_rng(14)
    m = Mirror(3, 200, 2, 96, 32)
    m.fill(g, [150, 0, 31])
    m.attend([1, 0, 1], _rand(g, 2, 4, 96, dtype="bf16"), "bf16", accumulate=True)
    other = KVCache(4, 333, 2, 96, block_tokens=32)
    for s in range(3):
        state = m.cache.export(s)
        if state[0].shape[1]:
            other.load(3 - s, *state)                                           # host arrays
            other.load(3 - s, *[torch.from_numpy(a).cuda() for a in state])     # device arrays
            for a, b in zip(state, other.export(3 - s)):
                assert np.array_equal(a, b)
    assert other.lengths.tolist() == [0, 31, 0, 150]


# ---- refusals ----------------------------------------------------------------


def test_refusals():
    from vicinity_b200 import KVCache, Rotary

    c = KVCache(2, 100, 2, 64, block_tokens=16)
    bf = dict(dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(5, 2, 64, **bf)
    q = torch.zeros(5, 4, 64, **bf)
    with pytest.raises(ValueError, match="capacity"):
        c.append(torch.zeros(101, 2, 64, **bf), torch.zeros(101, 2, 64, **bf), [101, 0])
    assert c.lengths.tolist() == [0, 0]
    with pytest.raises(ValueError, match="one entry"):
        c.append(k, k, [5])
    with pytest.raises(ValueError, match="must not be negative"):
        c.append(k, k, [6, -1])
    with pytest.raises(ValueError, match=r"k must be \[4"):
        c.append(k, k, [4, 0])
    with pytest.raises(ValueError, match="key/value heads"):
        c.append(torch.zeros(5, 1, 64, **bf), torch.zeros(5, 1, 64, **bf), [5, 0])
    with pytest.raises(ValueError, match="element type"):
        c.append(k, k.half(), [5, 0])
    with pytest.raises(ValueError, match="device memory"):
        c.append(k.cpu(), k.cpu(), [5, 0])
    with pytest.raises(ValueError, match="contiguous in its last"):
        c.append(torch.zeros(5, 2, 128, **bf)[..., ::2], k, [5, 0])
    c.append(k, k, [5, 0])
    with pytest.raises(ValueError, match="truncated"):
        c.truncate([6, 0])
    with pytest.raises(ValueError, match="multiple"):
        c.attend(torch.zeros(1, 3, 64, **bf), [1, 0], torch.zeros(1, 3, 64, **bf))
    with pytest.raises(ValueError, match="unsupported"):
        c.attend(q.float(), [5, 0], q.float())
    with pytest.raises(ValueError, match="heads of q"):
        c.attend(q, [5, 0], torch.zeros(5, 2, 64, **bf))
    with pytest.raises(ValueError, match="must not overlap"):
        c.attend(q, [5, 0], torch.zeros(5, 1, 64, **bf).expand(5, 4, 64))
    with pytest.raises(ValueError, match="finite"):
        c.attend(q, [5, 0], q.clone(), scale=math.inf)
    with pytest.raises(ValueError, match="lse"):
        c.attend(q, [5, 0], q.clone(), lse=torch.zeros(5, 3, device="cuda"))
    with pytest.raises(ValueError, match="twice"):
        c.evict([0], [0], 4, 1)
    with pytest.raises(ValueError, match="budget"):
        c.evict([0], [1], 101, 1)
    with pytest.raises(ValueError, match="recent"):
        c.evict([0], [1], 4, 5)
    with pytest.raises(ValueError, match="below 2"):
        c.evict([0], [2], 4, 1)
    with pytest.raises(ValueError, match="holds only"):
        c.read([3, 0], [3, 0], k[:3].clone(), k[:3].clone())
    with pytest.raises(ValueError, match="kept"):
        c.evict([0], [1], 4, 1, kept=torch.zeros(1, 2, 3, dtype=torch.int32, device="cuda"))
    r = Rotary(32)
    with pytest.raises(ValueError, match="at least the rotated"):
        r.apply(torch.arange(5).cuda(), torch.zeros(5, 2, 16, **bf))
    with pytest.raises(ValueError, match="int64"):
        r.apply(torch.arange(5, dtype=torch.int32).cuda(), q)
    with pytest.raises(ValueError, match="out_k without k"):
        r.apply(torch.arange(5).cuda(), q, out_k=k)
    with pytest.raises(ValueError, match="heads of its input"):
        r.apply(torch.arange(5).cuda(), q, out_q=torch.zeros(5, 2, 64, **bf))
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="captured"):
        with torch.cuda.graph(graph, stream=s):
            c.attend(q, [5, 0], q.clone(), stream=torch.cuda.current_stream().cuda_stream)
    # nothing above changed the cache
    assert c.lengths.tolist() == [5, 0]


def test_empty_calls():
    from vicinity_b200 import KVCache, Rotary

    c = KVCache(2, 100, 2, 64)
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    c.append(none, none, [0, 0])
    c.attend(none, [0, 0], none)
    c.read([0, 0], [0, 0], none, none)
    c.evict([], [], 4, 1)
    c.evict([0], [1], 4, 1)
    Rotary(64).apply(torch.zeros(0, dtype=torch.int64, device="cuda"), none)
    assert c.lengths.tolist() == [0, 0]


@pytest.mark.parametrize("seqs", [16, 17, 40, 300])
def test_many_sequences(seqs):
    # plans of up to 16 and of up to 256 sequences, and more than one plan;
    # some sequences take no part, and the rows of the others still line up
    g = np.random.default_rng(seqs)
    m = Mirror(2 * seqs, 48, 1, 32, 16)
    m.fill(g, [int(c) for c in g.integers(0, 40, seqs)] + [0] * seqs)
    counts = [int(c) for c in g.integers(0, 4, 2 * seqs)]
    m.fill(g, counts)
    m.check()
    q = _rand(g, sum(counts), 2, 32, dtype="bf16")
    m.attend(counts, q, "bf16", accumulate=True)
    more = [int(c) for c in g.choice([0, 1, 20], 2 * seqs)]      # both attention kernels in one call
    m.attend(more, _rand(g, sum(more), 2, 32, dtype="f16"), "f16", accumulate=True)
    kept = torch.empty(seqs, 1, 9, dtype=torch.int32, device="cuda")
    lens = m.cache.lengths.tolist()
    m.cache.evict(list(range(seqs)), list(range(seqs, 2 * seqs)), 9, 2, kept=kept)
    for s in range(seqs):
        at = ref.keep(m.w[s][0], lens[s], 9, 2)
        assert np.array_equal(kept[s, 0].cpu().numpy(), np.pad(at, (0, 9 - len(at)), constant_values=-1))
        m.k[seqs + s][0], m.v[seqs + s][0] = m.k[s][0].kept(at), m.v[s][0].kept(at)
    m.check()
    lens = m.cache.lengths.tolist()
    k, v = (torch.empty(sum(lens), 1, 32, dtype=torch.float32, device="cuda") for _ in range(2))
    m.cache.read([0] * (2 * seqs), lens, k, v)
    assert np.array_equal(_np(k)[:, 0], np.concatenate([h[0].values() for h in m.k]))
    assert np.array_equal(_np(v)[:, 0], np.concatenate([h[0].values() for h in m.v]))


def test_streaming_example_runs_them_together():
    import importlib.util

    from tests.conftest import ROOT

    spec = importlib.util.spec_from_file_location("kv_cache_stream", ROOT / "examples" / "kv_cache_stream.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    # nothing evicted: the outputs differ by the 8-bit codes alone
    assert example.main(["--prompt", "300", "--steps", "20", "--budget", "600"]) > 0.999
    # cut down to a quarter: most of the attention is left
    assert example.main(["--prompt", "1500", "--steps", "60", "--budget", "400"]) > 0.5


@pytest.mark.parametrize("which", ["keys", "values"])
def test_attend_poisoned_keys_or_values_alone(which):
    # NaN keys make the row NaN, its lse and the weights it gives too; NaN
    # values the row's output only
    g = np.random.default_rng(20)
    for counts in ([1, 1], [30, 50], [200, 1]):
        m = Mirror(2, 640, 1, 64, 16)
        m.fill(g, [150, 96])
        good = _rand(g, 32, 1, 64, dtype="f32")
        bad = torch.full((32, 1, 64), math.nan, device="cuda")
        m.append([16, 16], bad if which == "keys" else good, good if which == "keys" else bad)
        m.fill(g, counts)
        q = _rand(g, sum(counts), 4, 64, dtype="bf16")
        m.attend(counts, q, "bf16", accumulate=True)
        m.attend(counts, q, "bf16", causal=False)


def test_weights_without_stored_scores():
    # the scores of 16 rows over 2.2 million tokens of 8 heads (1.1 GB) are not
    # kept but computed again: the same weights as from two halves of the rows
    from vicinity_b200 import KVCache

    n, heads, d = 2_200_000, 8, 32
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = KVCache(1, n, heads, d, block_tokens=128)
    k = torch.randn(n, heads, d, generator=g, device="cuda").to(torch.bfloat16)
    cache.append(k, k, [n])
    del k
    q = torch.randn(1, heads, 16, d, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.as_tensor(cache.weights, device="cuda")
    out = torch.empty(1, heads * 16, d, dtype=torch.bfloat16, device="cuda")
    cache.attend(q.view(1, -1, d), [1], out, accumulate=True)
    whole = w[0].clone()
    w.zero_()
    halves = []
    for part in (q[:, :, :8], q[:, :, 8:]):
        o = torch.empty(1, heads * 8, d, dtype=torch.bfloat16, device="cuda")
        cache.attend(part.reshape(1, -1, d), [1], o, accumulate=True)
        halves.append(o.view(1, heads, 8, d))
    # scores up to about 30 in binary logarithms: |err| <= 2 (d + 16) u 30 + 64 u 22, each way
    rel = 2 * (2 * (d + 16) * U * 30 + 64 * U * 22)
    assert ((whole - w[0]).abs() <= rel * w[0] + 1e-12).all()
    assert abs(float(whole.double().sum()) - heads * 16) <= 1e-2
    assert torch.allclose(out.view(1, heads, 16, d).float(), torch.cat(halves, 2).float(), rtol=2.0 ** -7, atol=1e-6)


def test_rotary_wide_heads():
    # one pair of a very wide head, many heads: the largest items per CTA
    from vicinity_b200 import Rotary

    g = np.random.default_rng(21)
    q = _rand(g, 600, 70, 4096, dtype="bf16")
    r = Rotary(2)
    pos = torch.arange(600).cuda()
    out = torch.empty_like(q)
    r.apply(pos, q, out_q=out)
    assert torch.equal(out[..., 2:], q[..., 2:])
    want = ref.rotary(_np(q[..., :2]), np.arange(600), r.frequencies())
    assert (np.abs(_np(out[..., :2]) - want) <= _rotary_bound(q[..., :2], want, r.frequencies(), False, 1.0, "bf16")).all()
    with pytest.raises(ValueError, match="at most 4096"):
        r.apply(pos[:1], torch.zeros(1, 1, 4104, device="cuda"))


# ---- the whole range of scales ------------------------------------------------


def _attention64(q, k, v, causal, scale):
    """q [n, g, d] over k, v [len, d] of one head, in 64 bits on the GPU: (out, lse, weights, sum p |v|, max scale sum |q k|)."""
    n, L = q.shape[0], k.shape[0]
    q, k, v = q.double(), k.double(), v.double()
    s = scale * torch.einsum("ngd,ld->ngl", q, k)
    if causal:
        seen = torch.arange(L, device="cuda") < L - n + 1 + torch.arange(n, device="cuda")[:, None]
        s = torch.where(seen[:, None], s, -math.inf)
    p = torch.softmax(s, -1)
    top = abs(scale) * torch.einsum("ngd,ld->ngl", q.abs(), k.abs()).amax(-1)
    return p @ v, torch.logsumexp(s, -1), p.sum((0, 1)), p @ v.abs(), top


# queries times query heads per key/value head: both forms of the decoding
# kernel, one row tile, two
ROWS = [(1, 2), (3, 5), (20, 3), (150, 1)]


@pytest.mark.parametrize("n,group", ROWS)
@pytest.mark.parametrize("causal", [True, False])
def test_attend_zero_keys_and_values_over_a_long_sequence(n, group, causal):
    # equal scores: lse is the logarithm of the tokens seen and each gets the
    # same weight, whatever scale a block of zeros has
    from vicinity_b200 import KVCache

    L, d = 200_000, 32
    cache = KVCache(1, L, 1, d, block_tokens=128)
    zero = torch.zeros(L, 1, d, dtype=torch.bfloat16, device="cuda")
    cache.append(zero, zero, [L])
    q = torch.randn(n, group, d, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(torch.bfloat16)
    out, lse = torch.full_like(q, 7.0), torch.empty(n, group, device="cuda")
    cache.attend(q, [n], out, lse=lse, causal=causal, accumulate=True)
    w = torch.as_tensor(cache.weights, device="cuda")[0, 0, :L].double()
    seen = (L - n + 1 + torch.arange(n, device="cuda") if causal else torch.full((n,), L, device="cuda")).double()
    assert (out == 0).all()
    assert ((lse.double() - seen.log()[:, None]).abs() <= 16 * U * (1 + math.log(L))).all()
    each = (torch.arange(L, device="cuda") < seen[:, None]).double() / seen[:, None]
    want = group * each.sum(0)
    assert ((w - want).abs() <= (32 * U * (1 + math.log(L)) + 4 * U) * want).all()


@pytest.mark.parametrize("n,group", ROWS)
@pytest.mark.parametrize("zeros_first", [True, False])
def test_attend_a_long_run_of_zeros_beside_values(n, group, zeros_first):
    from vicinity_b200 import KVCache

    Z, V, d = 70_000, 700, 64
    g = torch.Generator(device="cuda").manual_seed(6)
    cache = KVCache(1, Z + V, 1, d, block_tokens=16)
    zero = torch.zeros(Z, 1, d, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.randn(V, 1, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    for a, b in [(zero, zero), (k, v)] if zeros_first else [(k, v), (zero, zero)]:
        cache.append(a, b, [a.shape[0]])
    q = (2 * torch.randn(n, group, d, generator=g, device="cuda")).to(torch.bfloat16)
    out, lse = torch.full_like(q, 7.0), torch.empty(n, group, device="cuda")
    cache.attend(q, [n], out, lse=lse, accumulate=True)
    w = torch.as_tensor(cache.weights, device="cuda")[0, 0, :Z + V].double()
    kk, vv = (torch.empty(Z + V, 1, d, device="cuda") for _ in range(2))
    cache.read([0], [Z + V], kk, vv)
    want, want_lse, want_w, size, top = _attention64(q, kk[:, 0], vv[:, 0], True, d ** -0.5)
    e = (d + 16) * U * top
    assert ((lse.double() - want_lse).abs() <= e + 16 * U * (1 + want_lse.abs())).all()
    soft = 2 * e + 32 * U * (1 + want_lse.abs())
    tol = 1.01 * ROUND["bf16"] * want.abs() + (2.0 ** -11 + soft)[..., None] * size
    tol += (Z + V) * 2.0 ** -36 * float(vv.abs().max())
    assert ((out.double() - want).abs() <= tol).all()
    assert ((w - want_w).abs() <= (soft.max() + 4 * U) * want_w + 1e-12).all()


@pytest.mark.parametrize("n,group", ROWS)
@pytest.mark.parametrize("length", [200, 3000])
def test_attend_values_of_all_magnitudes(length, n, group):
    # runs of tokens whose values are 0, or up to 2^120 apart, with keys of one
    # magnitude: the denominators do not depend on the values
    g = np.random.default_rng(length + n)
    for sizes in ([0.0, 2.0 ** 60], [2.0 ** 60, 0.0], [2.0 ** 100, 2.0 ** -90, 1.0, 0.0],
                  [0.0, 2.0 ** 20, 0.0, 2.0 ** 110, 2.0 ** -110], [2.0 ** -95], [2.0 ** 118, 0.0, 2.0 ** -60]):
        m = Mirror(1, length, 1, 64, 16)
        ends = [length * (i + 1) // len(sizes) for i in range(len(sizes))]
        for a, b, size in zip([0] + ends, ends, sizes):
            m.append([b - a], _rand(g, b - a, 1, 64, dtype="bf16"), _rand(g, b - a, 1, 64, dtype="bf16", scale=size))
        q = _rand(g, n, group, 64, dtype="bf16", scale=2.0)
        m.attend([n], q, "bf16", accumulate=True)
        m.attend([n], q, "bf16", causal=False)


@pytest.mark.parametrize("n,group", ROWS)
def test_attend_a_long_run_of_zeros_within_a_chunk(n, group):
    # as many heads as CTAs run at once, so that none is cut: a CTA's own sums
    # pass 32,768 tokens of zeros before the values come
    from vicinity_b200 import KVCache

    Z, V, d, heads = 39_000, 300, 32, 296
    g = torch.Generator(device="cuda").manual_seed(7)
    cache = KVCache(1, Z + V, heads, d, block_tokens=64)
    zero = torch.zeros(1, 1, d, dtype=torch.bfloat16, device="cuda").expand(Z, heads, d)
    cache.append(zero, zero, [Z])
    k, v = (torch.randn(V, heads, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    cache.append(k, v, [V])
    q = torch.randn(n, heads * group, d, generator=g, device="cuda").to(torch.bfloat16)
    out, lse = torch.full_like(q, 7.0), torch.empty(n, heads * group, device="cuda")
    cache.attend(q, [n], out, lse=lse)
    kk, vv = (torch.empty(Z + V, heads, d, device="cuda") for _ in range(2))
    cache.read([0], [Z + V], kk, vv)
    for h in (0, 100, 295):
        at = slice(h * group, (h + 1) * group)
        want, want_lse, _, size, top = _attention64(q[:, at], kk[:, h], vv[:, h], True, d ** -0.5)
        e = (d + 16) * U * top
        assert ((lse[:, at].double() - want_lse).abs() <= e + 16 * U * (1 + want_lse.abs())).all()
        tol = 1.01 * ROUND["bf16"] * want.abs() + (2.0 ** -11 + 2 * e + 32 * U * (1 + want_lse.abs()))[..., None] * size
        tol += (Z + V) * 2.0 ** -36 * float(vv.abs().max())
        assert ((out[:, at].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("n,group", ROWS)
def test_attend_largest_keys_smallest_queries(n, group):
    # keys near the largest scale and queries near the smallest numbers: their
    # scores are ordinary, in the attention and in the weights
    g = np.random.default_rng(30 + n)
    m = Mirror(1, 400, 2, 64, 32)
    for size in (124, 100, 124):
        m.append([130], _rand(g, 130, 2, 64, dtype="bf16", scale=2.0 ** size), _rand(g, 130, 2, 64, dtype="bf16"))
    q = _rand(g, n, 2 * group, 64, dtype="bf16", scale=2.0 ** -122)
    m.attend([n], q, "bf16", accumulate=True)


@pytest.mark.parametrize("where", ["host", "device"])
def test_load_refuses_scales_that_are_none(where):
    # scales are powers of two in [2^-100, 2^120], or NaN
    from vicinity_b200 import KVCache

    g = np.random.default_rng(31)
    c = KVCache(2, 100, 2, 32, block_tokens=16)

    def load(ks, vs):
        a = [g.integers(-127, 128, (2, 70, 32)).astype(np.int8), ks, g.integers(-127, 128, (2, 70, 32)).astype(np.int8), vs]
        c.load(0, *(a if where == "host" else [torch.from_numpy(x).cuda() for x in a]))

    good = np.float32(2.0) ** g.integers(-100, 121, (2, 5)).astype(np.float32)
    good[0, 0], good[0, 1], good[1, 4] = 2.0 ** -100, 2.0 ** 120, np.nan
    load(good, good[::-1].copy())
    before = c.export(0)
    for bad in (0.0, -0.0, -1.0, 3.0, 1.0 / 127, 2.0 ** -101, 2.0 ** 121, 2.0 ** -130, math.inf, -math.inf,
                float(np.nextafter(np.float32(1), np.float32(2)))):
        for at in ((0, 0), (1, 4)):
            scales = good.copy()
            scales[at] = bad
            for pair in ((scales, good), (good, scales)):
                with pytest.raises(ValueError, match="scales"):
                    load(*pair)
    assert c.lengths.tolist() == [70, 0]
    for a, b in zip(before, c.export(0)):
        assert np.array_equal(a, b, equal_nan=a.dtype == np.float32)


def test_misaligned_addresses_are_refused():
    # through the C entry points: an array must lie on a multiple of its element
    import ctypes as C

    from vicinity_b200 import KVCache, Rotary, _lib

    lib, bad = _lib.load(), _lib.VG_ERR_INVALID_PARAMETER
    c = KVCache(2, 64, 1, 32, block_tokens=16)
    k = torch.zeros(5, 1, 32, dtype=torch.bfloat16, device="cuda")
    c.append(k, k, [5, 0])
    room = torch.zeros(64, dtype=torch.int64, device="cuda")
    counts, src, dst = ((C.c_uint32 * n)(*x) for n, x in ((2, (5, 0)), (1, (0,)), (1, (1,))))
    at = lambda x: (C.c_int64 * 4)(x, 1, 32, 32)  # noqa: E731
    q, out = at(k.data_ptr()), at(k.clone().data_ptr())
    for off in (1, 2, 3):
        assert lib.vg_kv_attend(c._h, counts, _lib.BF16, q, out, room.data_ptr() + off, 1.0, 0, None) == bad
        assert "lse" in _lib.last_error()
        assert lib.vg_kv_evict(c._h, 1, src, dst, 4, 1, room.data_ptr() + off, None) == bad
        assert "kept" in _lib.last_error()
    r = Rotary(32)
    for off in (1, 2, 4, 7):
        assert lib.vg_rotary_apply(r._h, _lib.BF16, 32, room.data_ptr() + off, 5, q, out, None, None, 0, 0, None) == bad
        assert "positions" in _lib.last_error()
    odd = at(k.data_ptr() + 1)
    assert lib.vg_kv_append(c._h, counts, _lib.BF16, odd, q, None) == bad
    assert c.lengths.tolist() == [5, 0]


def test_growing_sequences_need_no_new_memory():
    # a decoding loop with weights: lengths pass multiples of 16 and of the
    # chunks, the working memory stays what the first step took
    g = np.random.default_rng(33)
    m = Mirror(5, 1500, 2, 64, 32)
    m.fill(g, [900, 13, 0, 601, 310])
    before = None
    for _ in range(150):
        k = _rand(g, 5, 2, 64, dtype="bf16")
        m.cache.append(k, k, [1] * 5)
        q = _rand(g, 5, 8, 64, dtype="bf16")
        m.cache.attend(q, [1] * 5, torch.empty_like(q), accumulate=True)
        now = int(m.cache.info().device_bytes)
        assert before in (None, now)
        before = now


def test_growing_prompts_need_new_memory_rarely():
    # chunks of a prompt against all before them: working memory at least doubles where it grows
    g = np.random.default_rng(34)
    m = Mirror(2, 6000, 2, 64, 64)
    q = _rand(g, 200, 4, 64, dtype="bf16")
    held = [int(m.cache.info().device_bytes)]
    for step in range(29):
        counts = [100, 100] if step % 2 else [200, 0]
        k = _rand(g, 200, 2, 64, dtype="bf16")
        m.cache.append(k, k, counts)
        m.cache.attend(q, counts, torch.empty_like(q), accumulate=True)
        held.append(int(m.cache.info().device_bytes))
    # one step in which every buffer is made, and a doubling of the partial sums' at most every other length
    assert len(set(held)) <= 7, sorted(set(held))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rot", [(128, 128), (96, 64), (50, 26)])
def test_rotary_in_place_within_a_fused_tensor(d, rot, layout):
    # queries and keys as slices of one projection, rotated where they lie
    from vicinity_b200 import Rotary

    g = np.random.default_rng(37)
    t = 3001
    x = _rand(g, t, 7, d, dtype="bf16")
    pos = torch.arange(5, 5 + t).cuda()
    r = Rotary(rot, layout=layout)
    want = x.clone()
    r.apply(pos, x[:, :4], x[:, 4:6], out_q=want[:, :4], out_k=want[:, 4:6])
    r.apply(pos, x[:, :4], x[:, 4:6])
    assert torch.equal(x, want)


def test_attend_in_place():
    # out may be q, in every form of the kernels
    from vicinity_b200 import KVCache

    g = np.random.default_rng(35)
    m = Mirror(4, 3000, 2, 64, 32)
    m.fill(g, [3000, 40, 700, 500])
    for counts in ([1, 1, 1, 1], [4, 0, 16, 1], [20, 300, 1, 64]):
        q = _rand(g, sum(counts), 8, 64, dtype="bf16")
        want, w = torch.empty_like(q), torch.as_tensor(m.cache.weights, device="cuda")
        w.zero_()
        m.cache.attend(q, counts, want, accumulate=True)
        want_w = w.clone()
        w.zero_()
        m.cache.attend(q, counts, q, accumulate=True)
        assert torch.equal(q, want) and torch.equal(w, want_w)
    # the same memory in another order is refused
    q = _rand(g, 8, 8, 64, dtype="bf16")
    with pytest.raises(ValueError, match="strides of q"):
        m.cache.attend(q, [2] * 4, q.transpose(0, 1))
    # more scores than are kept: they are computed again from the queries
    n, heads, d = 2_200_000, 8, 32
    gen = torch.Generator(device="cuda").manual_seed(4)
    cache = KVCache(1, n, heads, d, block_tokens=128)
    k = torch.randn(n, heads, d, generator=gen, device="cuda").to(torch.bfloat16)
    cache.append(k, k, [n])
    del k
    q = torch.randn(1, heads * 16, d, generator=gen, device="cuda").to(torch.bfloat16)
    want, w = torch.empty_like(q), torch.as_tensor(cache.weights, device="cuda")
    cache.attend(q, [1], want, accumulate=True)
    want_w = w.clone()
    w.zero_()
    cache.attend(q, [1], q, accumulate=True)
    assert torch.equal(q, want) and torch.equal(w, want_w)


def test_weights_are_ordered_across_streams():
    # each call on a stream of its own, appends, attention and eviction: the
    # state is that of the same calls on one stream, bit for bit
    g = np.random.default_rng(36)
    one, many = (Mirror(4, 4000, 2, 128, 64) for _ in range(2))
    lens = [3600, 1, 777, 0]
    n = sum(lens)
    k, v = (_rand(g, n, 2, 128, dtype="bf16") for _ in range(2))
    more = [_rand(g, 40 * 3, 2, 128, dtype="bf16") for _ in range(6)]
    queries = [_rand(g, 3 * c, 8, 128, dtype="bf16") for c in (1, 100, 2, 1, 40, 1)]
    outs = [[torch.empty_like(q) for q in queries] for _ in range(2)]
    torch.cuda.synchronize()
    for m, out, streams in ((one, outs[0], None), (many, outs[1], [torch.cuda.Stream() for _ in range(20)])):
        at = iter(streams) if streams else None
        stream = (lambda: next(at).cuda_stream) if streams else (lambda: None)
        m.cache.append(k, v, lens, stream=stream())
        for x, q, o in zip(more, queries, out):
            m.cache.append(x, x, [40] * 3 + [0], stream=stream())
            m.cache.attend(q, [q.shape[0] // 3] * 3 + [0], o, accumulate=True, stream=stream())
        total = torch.as_tensor(m.cache.weights, device="cuda")
        m.cache.evict([0], [3], 700, 50, stream=stream())
        torch.cuda.synchronize()
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    lengths = one.cache.lengths
    assert lengths.tolist() == many.cache.lengths.tolist() == [3840, 241, 1017, 700]
    for s in range(4):
        for a, b in zip(one.cache.export(s), many.cache.export(s)):
            assert np.array_equal(a, b)
    # every query gives each of its heads' tokens one unit in all, within the
    # weights' bound: 2 (d + 16) u 10 + 32 u 10 for scores of sum |q k| below 10
    # (a query that sees no token gives nothing)
    for s in range(3):
        rows = 4 * sum(min(q.shape[0] // 3, lens[s] + 40 * (i + 1)) for i, q in enumerate(queries))
        w = total[s, :, :int(lengths[s])].double().sum(-1)
        assert ((w - rows).abs() <= rows * 2.5e-4).all()


def test_load_and_export_of_rows_past_2_gb():
    # a head's codes lie further apart than a strided copy reaches
    from vicinity_b200 import KVCache

    g = np.random.default_rng(38)
    small, large = (KVCache(2, cap, 2, 128, block_tokens=64) for cap in (500, (1 << 24) + 100))
    k = _rand(g, 300, 2, 128, dtype="bf16")
    for c in (small, large):
        c.append(k, k, [0, 300])
    q = _rand(g, 1, 4, 128, dtype="bf16")
    for c in (small, large):
        c.attend(q, [0, 1], torch.empty_like(q), accumulate=True)
    state = small.export(1)
    for a, b in zip(state, large.export(1)):
        assert np.array_equal(a, b)
    large.load(0, *state)
    for a, b in zip(state, large.export(0)):
        assert np.array_equal(a, b)
    large.load(0, *state[:4])      # without weights: zeros
    assert not large.export(0)[4].any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,group", ROWS)
def test_attend_a_single_token_gives_its_value(n, group, dtype):
    # the largest probability of a row is not rounded: a query that sees one
    # token gets its value, code times scale, to the last bit
    from vicinity_b200 import KVCache

    g = np.random.default_rng(39 + n)
    cache = KVCache(1, n, 2, 64, block_tokens=16)
    k, v = (_rand(g, n, 2, 64, dtype="bf16", scale=s) for s in (3.0, 0.3))
    q = _rand(g, n, 2 * group, 64, dtype=dtype, scale=2.0)
    for length in (1, n):      # the first query of a prompt sees the first token alone
        cache.truncate([0])
        cache.append(k[:length], v[:length], [length])
        kk, vv = (torch.empty(length, 2, 64, dtype=q.dtype, device="cuda") for _ in range(2))
        cache.read([0], [length], kk, vv)
        out = torch.full_like(q, 7.0)
        cache.attend(q, [n], out)
        row = n - length       # those before it see nothing
        assert torch.equal(out[row], vv[0].repeat_interleave(group, 0))


@pytest.mark.parametrize("n,group", ROWS)
@pytest.mark.parametrize("size", [5, 12, 20, 50])
def test_attend_very_large_scores(size, n, group):
    # scores of 2^(2 size + 3), up to far more than f32 resolves to whole numbers:
    # tokens that tie for the largest share the attention, others get none.
    # Everything is a power of two, so the scores are exact and add nothing to
    # the bounds, which are those of small scores.
    from vicinity_b200 import KVCache

    g = np.random.default_rng(40 + size)
    L, d = 3000, 64
    sign = np.where(g.random((1, 1, d)) < 0.5, -1.0, 1.0)
    k = np.where(g.random((L, 1, d)) < 0.5, -1.0, 1.0) * 2.0 ** size     # far below the ties, below
    k[7::64] = -2 * sign * 2.0 ** size                                      # every other block has another scale
    tie = np.setdiff1d(g.choice(L, 40, replace=False), np.arange(7, L, 64))
    k[tie] = sign * 2.0 ** size
    v = g.standard_normal((L, 1, d))
    v[:L // 4] *= 2.0 ** 30
    v[L // 4:L // 2] = 0.0
    v[L // 2:3 * L // 4] *= 2.0 ** -40
    q = np.broadcast_to(sign * 2.0 ** size, (n, group, d)) * 2.0 ** -(np.arange(n) % 3)[:, None, None]
    kt, vt, qt = (torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16).cuda() for x in (k, v, q))
    third = tie[(tie >= L // 2) & (tie < 3 * L // 4)]
    soft = 32 * U * (1 + math.log(L))
    for ties in (tie, tie[tie >= L // 2], third[:1]):
        for negative in (False, True):
            keys = kt.clone()
            keys[np.setdiff1d(tie, ties)] *= -1
            if negative:      # the ties' scores too, the others' further below
                keys = -4 * kt.abs() * torch.from_numpy(sign).to(kt)
                keys[ties] = -kt[ties]
            cache = KVCache(1, L, 1, d, block_tokens=32)
            cache.append(keys, vt, [L])
            kr, vr = (torch.empty(L, 1, d, device="cuda") for _ in range(2))
            cache.read([0], [L], kr, vr)
            assert torch.equal(kr, keys.float())
            want, want_lse, want_w, size_of, _ = _attention64(qt, kr[:, 0], vr[:, 0], False, 0.125)
            assert ((want_w > 0.9 * n * group / len(ties)).sum() == len(ties)) and want_w.sum() > (1 - 1e-9) * n * group
            out, lse = torch.full_like(qt, 7.0), torch.empty(n, group, device="cuda")
            cache.attend(qt, [n], out, lse=lse, scale=0.125, causal=False, accumulate=True)
            w = torch.as_tensor(cache.weights, device="cuda")[0, 0, :L].double()
            assert ((lse.double() - want_lse).abs() <= 16 * U * (1 + want_lse.abs())).all()
            tol = 1.01 * ROUND["bf16"] * want.abs() + (2.0 ** -11 + soft) * size_of
            tol += L * 2.0 ** -36 * float(vr[ties].abs().max())
            assert ((out.double() - want).abs() <= tol).all()
            assert ((w - want_w).abs() <= (soft + 4 * U) * want_w + 1e-12).all()


@pytest.mark.parametrize("n,group", ROWS)
@pytest.mark.parametrize("length", [300, 3000])
@pytest.mark.parametrize("huge", [80, 118])
def test_attend_tiny_values_beside_huge_ones_that_get_nothing(huge, length, n, group):
    # runs of tokens that no query looks at (2^-500 of the others' probability)
    # hold huge values: what is left of the tiny ones is not lost beside them
    g = torch.Generator(device="cuda").manual_seed(huge + length)
    from vicinity_b200 import KVCache

    for run in (16, 112, length // 32 * 16):     # whole blocks: no token shares a huge scale
        far = (torch.arange(length, device="cuda") // run % 2 == 1)
        for flip in (False, True):
            far = far ^ flip
            k = torch.randn(length, 1, 64, generator=g, device="cuda")
            k[..., 0] = torch.where(far, -200.0, 0.0)[:, None]
            v = torch.randn(length, 1, 64, generator=g, device="cuda")
            v *= torch.where(far, 2.0 ** huge, 2.0 ** -60)[:, None, None]
            q = torch.randn(n, group, 64, generator=g, device="cuda")
            q[..., 0] = 16.0
            k, v, q = (x.to(torch.bfloat16) for x in (k, v, q))
            cache = KVCache(1, length, 1, 64, block_tokens=16)
            cache.append(k, v, [length])
            kk, vv = (torch.empty(length, 1, 64, device="cuda") for _ in range(2))
            cache.read([0], [length], kk, vv)
            out, lse = torch.full_like(q, 7.0), torch.empty(n, group, device="cuda")
            cache.attend(q, [n], out, lse=lse, causal=False)
            want, want_lse, _, size, top = _attention64(q, kk[:, 0], vv[:, 0], False, 64 ** -0.5)
            e = (64 + 16) * U * top
            soft = 32 * U * (1 + want_lse.abs()) + 2 * e
            assert ((lse.double() - want_lse).abs() <= e + 16 * U * (1 + want_lse.abs())).all()
            tol = 1.01 * ROUND["bf16"] * want.abs() + (2.0 ** -11 + soft)[..., None] * size
            tol += length * 2.0 ** -36 * float(vv[~far].abs().max())
            assert ((out.double() - want).abs() <= tol).all()
