"""Cases of the key/value cache operators: rotary positions, appending to a cache
held in 8 bits, attention over it, and eviction by accumulated attention weight.

``own`` false computes an operator in its plain form (elementary torch
operations); ``own`` true calls the engine through its Python binding.

Formulas shared by every form:

* rotary: the pair (a, b) of frequency i at position p becomes
  m (a cos t - b sin t, a sin t + b cos t), t = p f_i; transposed (the gradient)
  with -sin.  Pairs are (2i, 2i + 1) or (i, i + r / 2); the head's dimensions from
  r on pass through.
* cache: tokens are held in blocks; per sequence, head and block one scale s for
  the keys and one for the values, the smallest power of two in
  [2^-100, 2^120] with 127 s >= every |x|, and codes round_half_even(x / s).  A block's
  scale only grows while tokens are appended to it; its codes are then rounded to
  the new scale.
* attention: softmax over the cached tokens a query sees, queries being the last
  tokens of the cache (token j of n sees the first len - n + j + 1); the weight of a
  cached token is the sum, over the queries and the heads that share it, of its
  probabilities, added to what the cache has accumulated.
* eviction: the `recent` newest tokens and those of largest weight (ties to the
  older one) up to `budget`, in order, in another sequence of the cache; a block's
  scale is the largest of its tokens' scales.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases ------------------------------------------------------------------


def listed():
    return [
        # one decode step of 16 sequences, positions deep in a long context
        dict(name="rotary step", op="rotary", tokens=16, start=90000, hq=32, hk=8, d=128, rot=128, layout="half",
             scaling="none", transpose=False, dtype="bf16"),
        # the gradient of a partly rotated head, adjacent pairs, odd sizes
        dict(name="rotary gradient", op="rotary", tokens=777, start=5, hq=12, hk=4, d=96, rot=64,
             layout="interleaved", scaling="linear", transpose=True, dtype="f32"),
        # a whole prompt with frequencies scaled for a context eight times as long
        dict(name="rotary prompt", op="rotary", tokens=16384, start=0, hq=32, hk=8, d=128, rot=128, layout="half",
             scaling="by_parts", transpose=False, dtype="bf16"),
        # one token for each of 16 sequences: most land inside a block that has tokens
        dict(name="append step", op="append", seqs=16, count=1, length=4100, spread=700, hk=8, d=128, block=64,
             dtype="bf16"),
        # two prompts, written in one call
        dict(name="append prompts", op="append", seqs=2, count=8192, length=0, spread=0, hk=8, d=128, block=64,
             dtype="bf16"),
        # one short sequence: what a call costs
        dict(name="attend short", op="attend", seqs=1, count=1, length=513, spread=0, hq=32, hk=8, d=128, block=64,
             weights=False, dtype="bf16"),
        # a serving batch of uneven lengths, one of them empty, that keeps weights for eviction
        dict(name="attend batch", op="attend", seqs=16, count=1, length=8192, spread=8192, hq=32, hk=8, d=128,
             block=64, weights=True, dtype="bf16"),
        # one very long sequence: the work is split over the tokens
        dict(name="attend long", op="attend", seqs=1, count=1, length=131101, spread=0, hq=32, hk=8, d=128, block=64,
             weights=False, dtype="bf16"),
        # a chunk of a long prompt against all that is cached before it, with weights
        dict(name="attend chunk", op="attend", seqs=1, count=1024, length=16384, spread=0, hq=32, hk=8, d=128,
             block=64, weights=True, dtype="bf16"),
        # a few tokens over the budget, small heads
        dict(name="evict few", op="evict", seqs=4, length=300, spread=40, budget=256, recent=32, hk=4, d=64,
             block=16),
        # sequences on both sides of the budget, odd sizes
        dict(name="evict uneven", op="evict", seqs=7, length=4999, spread=4700, budget=1001, recent=77, hk=5, d=96,
             block=32),
        # eight long prompts cut down before they are decoded
        dict(name="evict prompts", op="evict", seqs=8, length=16384, spread=0, budget=2048, recent=256, hk=8, d=128,
             block=64),
    ]


def draw(rng):
    def log(a, b):
        return min(b, max(a, round(math.exp(rng.uniform(math.log(a), math.log(b + 1))))))

    op = rng.choice(["rotary", "append", "attend", "attend", "evict"])
    d = rng.choice([64, 96, 128])
    hk = rng.choice([1, 2, 3, 5, 8])
    if op == "rotary":
        rot = rng.choice([d, d, d // 2])
        return dict(op=op, tokens=log(1, 8192), start=rng.randrange(100000), hq=hk * rng.choice([1, 2, 4]), hk=hk,
                    d=d, rot=rot, layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "by_parts"]), transpose=rng.random() < 0.3,
                    dtype=rng.choice(["f32", "f16", "bf16", "bf16"]))
    block = rng.choice([16, 32, 64, 64, 128])
    if op == "append":
        if rng.random() < 0.5:
            seqs, count = log(1, 64), rng.choice([1, 1, 2, 5])
        else:
            seqs, count = log(1, 4), log(6, 2500)
        length = log(1, 5000)
        return dict(op=op, seqs=seqs, count=count, length=length, spread=rng.randrange(length + 1), hk=hk, d=d,
                    block=block, dtype=rng.choice(["f32", "f16", "bf16", "bf16"]))
    if op == "attend":
        group = rng.choice([1, 2, 4, 4, 7, 8])
        if rng.random() < 0.65:
            seqs, count = log(1, 32), rng.choice([1, 1, 1, 2, 4])
            length = log(1, 131072 // seqs)
        else:
            seqs, count = log(1, 2), log(5, 500)
            length = count + log(1, 6000)
        length = max(length, count)
        return dict(op=op, seqs=seqs, count=count, length=length, spread=rng.randrange(length - count + 1), hq=hk * group,
                    hk=hk, d=d, block=block, weights=rng.random() < 0.5, dtype=rng.choice(["f16", "bf16", "bf16"]))
    length = log(40, 16384)
    budget = log(8, min(length, 4000))
    return dict(op=op, seqs=log(1, 8), length=length, spread=rng.randrange(length), budget=budget,
                recent=rng.randrange(budget + 1), hk=hk, d=d, block=block)


def lengths_of(case):
    """Tokens cached for each sequence before the call (for attention: its queries among them)."""
    n, top, spread = case["seqs"], case["length"], case["spread"]
    if n == 1 or spread == 0:
        return [top] * n
    step = 7 if n % 7 else 5 if n % 5 else 1
    return [top - (spread * ((i * step) % n)) // (n - 1) for i in range(n)]


def work(case):
    op = case["op"]
    if op == "rotary":
        values = case["tokens"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * values * BYTES[case["dtype"]] + 8 * case["tokens"], "flops": 4 * values}
    hk, d, block = case["hk"], case["d"], case["block"]
    lens = lengths_of(case)
    if op == "append":
        new = case["seqs"] * case["count"] * hk * d * 2
        held = sum(n % block for n in lens) * hk * d * 2  # read again only where the scale grows: not counted
        return {"bytes": new * (BYTES[case["dtype"]] + 1) + (new + held) * 3, "flops": 4 * new}
    if op == "attend":
        cached = sum(lens) * hk * d * 2 + sum(-(-n // block) for n in lens) * hk * 8
        rows = case["seqs"] * case["count"] * case["hq"]
        seen = sum(sum(max(0, n - case["count"] + j + 1) for j in range(case["count"])) for n in lens) * case["hq"]
        more = sum(lens) * hk * 8 if case["weights"] else 0
        return {"bytes": cached + rows * (2 * d * 2 + 4) + more, "flops": 4 * seen * d}
    kept = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": sum(lens) * hk * 4 + kept * hk * (2 * d * (1 + 1 + 1 + 2) + 8), "flops": kept * hk * 2 * d}


# ---- inputs -----------------------------------------------------------------


def frequencies(case):
    r, base = case["rot"], 10000.0
    f = [base ** (-2.0 * i / r) for i in range(r // 2)]
    if case["scaling"] == "linear":
        return [x / 4.0 for x in f], 1.0
    if case["scaling"] == "by_parts":
        def part(x):
            turns = 4096 * x / (2 * math.pi)
            g = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
            return (1 - g) * x / 8.0 + g * x
        return [part(x) for x in f], 0.1 * math.log(8.0) + 1.0
    return f, 1.0


def key_like(g, *shape):
    """Normal values with a few channels far larger than the others, as keys have."""
    x = torch.randn(*shape, generator=g, device="cuda")
    x[..., 3::41] *= 8.0
    return x


def scale_for(top):
    """The smallest power of two s in [2^-100, 2^120] with 127 s >= top."""
    m, e = torch.frexp(top)
    e = torch.where(top > 0, e - 7 + (m > 0.9921875).int(), -100)
    return torch.exp2(e.clamp(-100, 120).float())


def quantised(x, block):
    """Codes and block scales of [..., tokens, d] values (tokens a multiple of block)."""
    b = x.unflatten(-2, (-1, block))
    s = scale_for(b.abs().amax((-1, -2)))
    return torch.round(b / s[..., None, None]).to(torch.int8).flatten(-3, -2), s


def inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "rotary":
        t, dt = case["tokens"], DTYPES[case["dtype"]]
        f, m = frequencies(case)
        return dict(pos=case["start"] + torch.randperm(t, generator=g, device="cuda"),
                    q=torch.randn(t, case["hq"], case["d"], generator=g, device="cuda").to(dt),
                    k=key_like(g, t, case["hk"], case["d"]).to(dt),
                    f=torch.tensor(f, dtype=torch.float64, device="cuda"), m=m)
    n, hk, d, block = case["seqs"], case["hk"], case["d"], case["block"]
    lens = lengths_of(case)
    cap = -(-(max(lens) + (case["count"] if case["op"] == "append" else 0)) // block) * block
    at = torch.arange(cap, device="cuda")
    held = torch.tensor(lens, device="cuda")
    live = at < held[:, None]
    x = {"lens": held, "cap": cap}
    for name, make in (("k", key_like(g, n, hk, cap, d)), ("v", torch.randn(n, hk, cap, d, generator=g, device="cuda"))):
        make *= live[:, None, :, None]
        x[name + "c"], x[name + "s"] = quantised(make, block)
        del make
    if case["op"] == "append":
        t, dt = n * case["count"], DTYPES[case["dtype"]]
        x["k"] = (key_like(g, t, hk, d) * 1.3).to(dt)
        x["v"] = torch.randn(t, hk, d, generator=g, device="cuda").to(dt)
    elif case["op"] == "attend":
        x["q"] = torch.randn(n * case["count"], case["hq"], d, generator=g, device="cuda").to(DTYPES[case["dtype"]])
        x["w"] = torch.rand(n, hk, cap, generator=g, device="cuda") * live[:, None]
    else:
        # long-tailed weights, many of them equal (tokens that no query looked at)
        w = torch.rand(n, hk, cap, generator=g, device="cuda").pow(8).mul(16)
        x["w"] = torch.where(w < 0.01, torch.zeros(()).cuda(), w) * live[:, None]
    return x


def prepare(case, seed):
    x = inputs(case, seed)
    x["case"] = case
    op = case["op"]
    if op == "rotary":
        x["oq"], x["ok"] = torch.empty_like(x["q"]), torch.empty_like(x["k"])
        if own:
            from vicinity_b200 import Rotary

            scaled = {"none": {}, "linear": dict(factor=4.0),
                      "by_parts": dict(factor=8.0, original_length=4096, magnitude=x["m"])}[case["scaling"]]
            x["rotary"] = Rotary(case["rot"], base=10000.0, layout=case["layout"], scaling=case["scaling"], **scaled)
        return x
    n, hk, d, block, lens = case["seqs"], case["hk"], case["d"], case["block"], lengths_of(case)
    x["held"], x["each"] = lens, [case.get("count", 0)] * n
    if op == "append":
        # the tokens looked at after the call: from the start of the block that the first new one lands in
        starts = [a // block * block for a in lens]
        x["starts"], x["counts"] = starts, [a + case["count"] - s for a, s in zip(lens, starts)]
        first = torch.tensor(starts, device="cuda")
        width = -(-(case["count"] + block - 1) // block) * block
        slot = first[:, None] + torch.arange(width, device="cuda")
        x["first"], x["slot"] = first, slot
        x["within"] = (slot < (x["lens"] + case["count"])[:, None]).flatten().nonzero()[:, 0]
    elif op == "evict":
        x["starts"], x["counts"] = [0] * n, [min(a, case["budget"]) for a in lens]
        at = torch.arange(case["budget"], device="cuda")
        x["within"] = (at < x["lens"][:, None]).flatten().nonzero()[:, 0]
    if op == "attend":
        x["out"] = torch.empty_like(x["q"])
        x["lse"] = torch.empty(x["q"].shape[:2], device="cuda")
    else:
        rows = sum(x["counts"])
        x["kr"] = torch.empty(rows, hk, d, dtype=torch.bfloat16, device="cuda")
        x["vr"] = torch.empty_like(x["kr"])
    if own:
        from vicinity_b200 import KVCache

        more = n if op == "evict" else 0
        cache = KVCache(n + more, x["cap"], hk, d, block_tokens=block)
        for i, a in enumerate(lens):
            if a:
                nb = -(-a // block)
                cache.load(i, x["kc"][i, :, :a].contiguous(), x["ks"][i, :, :nb].contiguous(),
                           x["vc"][i, :, :a].contiguous(), x["vs"][i, :, :nb].contiguous(),
                           x["w"][i, :, :a].contiguous() if "w" in x else None)
        x["cache"] = cache
        x["weights"] = torch.as_tensor(cache.weights, device="cuda")
        if op == "evict":
            x["kept"] = torch.empty(n, hk, case["budget"], dtype=torch.int32, device="cuda")
            x["from"], x["to"] = list(range(n)), list(range(n, 2 * n))
            x["starts"], x["counts"] = [0] * (2 * n), [0] * n + x["counts"]
        for name in ("kc", "ks", "vc", "vs", "w"):
            x.pop(name, None)
    return x


# ---- one pass -----------------------------------------------------------------


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state, state["case"])


def own_rotary(x, case):
    x["rotary"].apply(x["pos"], x["q"], x["k"], out_q=x["oq"], out_k=x["ok"], transpose=case["transpose"])
    return {"q": x["oq"], "k": x["ok"]}


def own_append(x, case):
    x["cache"].truncate(x["held"])
    x["cache"].append(x["k"], x["v"], x["each"])
    x["cache"].read(x["starts"], x["counts"], x["kr"], x["vr"])
    return {"k": x["kr"], "v": x["vr"]}


def own_attend(x, case):
    x["cache"].attend(x["q"], x["each"], x["out"], lse=x["lse"], accumulate=case["weights"])
    w = {"w": x["weights"][:, :, :x["cap"]]} if case["weights"] else {}
    return {"out": x["out"], "lse": x["lse"], **w}


def own_evict(x, case):
    x["cache"].evict(x["from"], x["to"], case["budget"], case["recent"], kept=x["kept"])
    x["cache"].read(x["starts"], x["counts"], x["kr"], x["vr"])
    return {"kept": x["kept"], "k": x["kr"], "v": x["vr"], "w": x["weights"][case["seqs"]:, :, :case["budget"]]}


def plain_rotary(x, case):
    # the angle, and it alone, in 64 bits: in 32 an angle at position 10^5 is off by a hundredth
    t = x["pos"].double()[:, None] * x["f"]
    t = torch.remainder(t, 2 * math.pi).float()[:, None]
    c, s = torch.cos(t) * x["m"], torch.sin(t) * (-x["m"] if case["transpose"] else x["m"])
    return {name: plain_rotated(x[name], c, s, case) for name in ("q", "k")}


def plain_rotated(y, c, s, case):
    r, z = case["rot"], y.float()
    if case["layout"] == "half":
        a, b = z[..., :r // 2], z[..., r // 2:r]
        z = torch.cat([a * c - b * s, a * s + b * c, z[..., r:]], -1)
    else:
        a, b = z[..., 0:r:2], z[..., 1:r:2]
        z = torch.cat([torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2), z[..., r:]], -1)
    return z.to(y.dtype)


def plain_append(x, case):
    return {name: plain_appended(x[name], x[name + "c"], x[name + "s"], x, case) for name in ("k", "v")}


def plain_appended(new, codes, scales, x, case):
    n, count, block, hk, d = case["seqs"], case["count"], case["block"], case["hk"], case["d"]
    slot, width = x["slot"], x["slot"].shape[1]
    rows = slot.clamp(max=x["cap"] - 1)
    old = codes.gather(2, rows[:, None, :, None].expand(n, hk, width, d)).float()
    blocks = (slot[:, ::block] // block).clamp(max=scales.shape[2] - 1)
    s_old = scales.gather(2, blocks[:, None].expand(n, hk, -1))
    at = slot - x["lens"][:, None]
    is_new = (at >= 0) & (at < count)
    row = (torch.arange(n, device="cuda")[:, None] * count + at.clamp(0, count - 1)).flatten()
    fresh = new.index_select(0, row).float().view(n, width, hk, d).transpose(1, 2) * is_new[:, None, :, None]
    s = scale_for(fresh.unflatten(2, (-1, block)).abs().amax((-1, -2)))
    has_old = (slot[:, ::block] < x["lens"][:, None])[:, None]
    s_old = torch.where(has_old, s_old, torch.full_like(s_old, 2.0 ** -100))
    s = torch.maximum(s, s_old)
    each, each_old = s.repeat_interleave(block, 2)[..., None], s_old.repeat_interleave(block, 2)[..., None]
    code = torch.where(is_new[:, None, :, None], torch.round(fresh / each), torch.round(old * (each_old / each)))
    value = (code * each).to(torch.bfloat16).transpose(1, 2).reshape(n * width, hk, d)
    return value.index_select(0, x["within"])


def plain_attend(x, case):
    n, count, block, hk, d, cap = case["seqs"], case["count"], case["block"], case["hk"], case["d"], x["cap"]
    group = case["hq"] // hk
    k = x["kc"].float().unflatten(2, (-1, block)).mul_(x["ks"][..., None, None]).flatten(2, 3)
    q = x["q"].float().view(n, count, hk, group, d).permute(0, 2, 1, 3, 4).reshape(n, hk, count * group, d)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5)
    del k
    sees = x["lens"][:, None] - count + 1 + torch.arange(count, device="cuda")
    hidden = torch.arange(cap, device="cuda") >= sees[..., None]
    s.view(n, hk, count, group, cap).masked_fill_(hidden[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    w = {"w": x["w"].add_(p.sum(2))} if case["weights"] else {}
    v = x["vc"].float().unflatten(2, (-1, block)).mul_(x["vs"][..., None, None]).flatten(2, 3)
    out = torch.matmul(p, v).view(n, hk, count, group, d).permute(0, 2, 1, 3, 4)
    lse = (top + total.log())[..., 0].view(n, hk, count, group).permute(0, 2, 1, 3)
    return {"out": out.reshape(n * count, hk * group, d).to(x["q"].dtype),
            "lse": lse.reshape(n * count, hk * group).contiguous(), **w}


def plain_evict(x, case):
    n, hk, d, block, cap, budget = case["seqs"], case["hk"], case["d"], case["block"], x["cap"], case["budget"]
    at, held = torch.arange(cap, device="cuda"), x["lens"][:, None]
    key = torch.where((at >= held - case["recent"])[:, None], math.inf, x["w"])
    key = torch.where((at >= held)[:, None], -1.0, key)
    first = key.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    kept = torch.where(first < held[:, None], first, cap).sort(-1).values
    if kept.shape[2] < budget:
        kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[2]), value=cap)
    live, src = kept < cap, kept.clamp(max=cap - 1)
    w = torch.where(live, x["w"].gather(2, src), 0.0)
    pad = -budget % block
    out = {"kept": torch.where(live, kept, -1).int(), "w": w}
    for name in ("k", "v"):
        code = x[name + "c"].gather(2, src[..., None].expand(n, hk, budget, d)).float()
        s = torch.where(live, x[name + "s"].gather(2, src // block), 2.0 ** -100)
        top = torch.nn.functional.pad(s, (0, pad), value=2.0 ** -100).unflatten(2, (-1, block)).amax(-1)
        top = top.repeat_interleave(block, 2)[:, :, :budget]
        value = torch.round(code * (s / top)[..., None]) * top[..., None]
        rows = value.to(torch.bfloat16).transpose(1, 2).reshape(n * budget, hk, d)
        out[name] = rows.index_select(0, x["within"])
    return out


OWN = {"rotary": own_rotary, "append": own_append, "attend": own_attend, "evict": own_evict}
PLAIN = {"rotary": plain_rotary, "append": plain_append, "attend": plain_attend, "evict": plain_evict}


# ---- the definition in 64 bits ---------------------------------------------------


def exact(case, seed):
    x = inputs(case, seed)
    return {"rotary": exact_rotary, "append": exact_append, "attend": exact_attend, "evict": exact_evict}[case["op"]](x, case)


def exact_rotary(x, case):
    r, out = case["rot"], {}
    turn = torch.polar(torch.full((), x["m"], dtype=torch.float64, device="cuda"), x["pos"].double()[:, None] * x["f"])
    turn = (turn.conj() if case["transpose"] else turn)[:, None]
    for name in ("q", "k"):
        y = x[name].double()
        pairs = y[..., :r].unflatten(-1, (-1, 2) if case["layout"] == "interleaved" else (2, -1))
        pairs = pairs if case["layout"] == "interleaved" else pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z if case["layout"] == "interleaved" else z.transpose(-1, -2)
        y[..., :r] = z.flatten(-2)
        out[name] = y
    return out


def least_scale(top):
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -120) / 127)).clamp(-100, 120)
    e = torch.where(127 * torch.exp2(e - 1) >= top, e - 1, e)
    return torch.exp2(e.clamp(min=-100))


def exact_append(x, case):
    block, count, out = case["block"], case["count"], {"k": [], "v": []}
    for i, a in enumerate(lengths_of(case)):
        for name in ("k", "v"):
            first, end = a // block * block, a + count
            parts, new = [], x[name][i * count:(i + 1) * count].double().transpose(0, 1)
            for b in range(first, end, block):
                lo, hi = max(a, b), min(end, b + block)
                fresh = new[:, lo - a:hi - a]
                s = least_scale(fresh.abs().amax((1, 2)))[:, None, None]
                if b < a:
                    was = x[name + "s"][i, :, b // block].double()[:, None, None]
                    s = torch.maximum(s, was)
                    parts.append(torch.round(x[name + "c"][i, :, b:a].double() * was / s) * s)
                parts.append(torch.round(fresh / s) * s)
            out[name].append(torch.cat(parts, 1).transpose(0, 1))
    return {name: torch.cat(parts) for name, parts in out.items()}


def exact_attend(x, case):
    n, count, block, hk, d = case["seqs"], case["count"], case["block"], case["hk"], case["d"]
    group = case["hq"] // hk
    out = torch.zeros(n, count, case["hq"], d, dtype=torch.float64, device="cuda")
    lse = torch.full((n, count, case["hq"]), -math.inf, dtype=torch.float64, device="cuda")
    w = x["w"].double()
    for i, a in enumerate(lengths_of(case)):
        for h in range(hk if a else 0):
            k = (x["kc"][i, h].double().view(-1, block, d) * x["ks"][i, h].double()[:, None, None]).view(-1, d)[:a]
            v = (x["vc"][i, h].double().view(-1, block, d) * x["vs"][i, h].double()[:, None, None]).view(-1, d)[:a]
            heads = slice(h * group, (h + 1) * group)
            s = torch.einsum("tgd,ld->tgl", x["q"].view(n, count, -1, d)[i, :, heads].double(), k) / math.sqrt(d)
            last = torch.arange(a - count, a, device="cuda")[:, None, None]
            s = torch.where(torch.arange(a, device="cuda") <= last, s, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            out[i, :, heads], lse[i, :, heads] = torch.einsum("tgl,ld->tgd", p, v), torch.logsumexp(s, -1)
            w[i, h, :a] += p.sum((0, 1))
    got = {"out": out.flatten(0, 1), "lse": lse.flatten(0, 1)}
    return {**got, "w": w} if case["weights"] else got


def exact_evict(x, case):
    n, hk, d, block, budget = case["seqs"], case["hk"], case["d"], case["block"], case["budget"]
    kept = torch.full((n, hk, budget), -1, dtype=torch.int32, device="cuda")
    w = torch.zeros(n, hk, budget, dtype=torch.float64, device="cuda")
    out = {"k": [], "v": []}
    for i, a in enumerate(lengths_of(case)):
        m = min(a, budget)
        value = {name: torch.zeros(m, hk, d, dtype=torch.float64, device="cuda") for name in ("k", "v")}
        for h in range(hk):
            old = max(0, a - case["recent"])
            best = torch.argsort(-x["w"][i, h, :old].double(), stable=True)[:max(0, m - (a - old))]
            keep = torch.cat([best, torch.arange(max(old, a - m), a, device="cuda")]).sort().values
            kept[i, h, :m], w[i, h, :m] = keep.int(), x["w"][i, h, keep].double()
            for name in ("k", "v"):
                code, was = x[name + "c"][i, h, keep].double(), x[name + "s"][i, h, keep // block].double()
                top = torch.stack([c.amax() for c in was.split(block)]).repeat_interleave(block)[:m] if m else was
                value[name][:, h] = torch.round(code * (was / top)[:, None]) * top[:, None]
        for name in ("k", "v"):
            out[name].append(value[name])
    return {"kept": kept, "w": w, "k": torch.cat(out["k"]), "v": torch.cat(out["v"])}
