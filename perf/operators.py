"""The serving operators of a paged key/value cache, as calls to measure them on.

Four operators, as a decoding or prefilling program calls them between its matrix products:

``extend``   block tables, slots and positions of new tokens, from request lengths (``ops.paged_extend``)
``rotary``   rotary positions on queries and keys in the attention's layout (``ops.rotary``)
``append``   rotary positions on new tokens, their keys and values written into the pages (``ops.rotary_append``)
``attend``   attention of one new token per request over the pages (``ops.paged_attention``)

``listed()`` names twelve calls; ``draw`` gives further ones of the same ranges.  ``prepare`` makes what a
program holds before the call, ``run`` makes the call - with ``own`` through the package, without it in
elementary torch operations - ``work`` counts what the call cannot do without, ``exact`` gives its result
in 64 bits.

Page 0 of every cache is never given to a request, as allocators do that want a harmless default.
"""
from __future__ import annotations

import math

import torch

own = False

# The largest work of a drawn case, by operator: that of the largest listed one.
MOST_BYTES = {"extend": 1.1e6, "rotary": 1.7e8, "append": 2.1e8, "attend": 5.4e8}


def listed():
    return [
        # One decoding step of a full server: one token for each of 256 requests, one in sixteen needs a page.
        dict(name="extend_decode", op="extend", B=256, length=4000, new=1, ps=16),
        # A batch of prompts of unequal length enters, some behind a cached prefix: thousands of pages at once.
        dict(name="extend_prompts", op="extend", B=48, length=500, new=2500, ps=16),
        # Queries and keys of a grouped-query prefill, laid out by token as the projection leaves them.
        dict(name="rotary_prompt", op="rotary", B=4, S=2048, H=16, Hk=4, d=128, rot=128, dtype="bf16",
             interleaved=False, adjoint=False, base=10000.0, mscale=1.0, start=0),
        # The gradient through it for the smaller head: half of the head rotates, in neighbouring pairs, at
        # positions far into a long context with stretched frequencies; an odd length.
        dict(name="rotary_adjoint", op="rotary", B=3, S=1777, H=16, Hk=16, d=64, rot=32, dtype="fp16",
             interleaved=True, adjoint=True, base=500000.0, mscale=1.25, start=900000),
        # The new tokens of a decoding step on their way into the cache.
        dict(name="append_decode", op="append", T=64, H=32, Hk=8, d=128, rot=128, ps=16, dtype="bf16",
             interleaved=False, base=10000.0, mscale=1.0, start=3000),
        # The tokens of several prompts, packed one behind the other and padded at the end.
        dict(name="append_prompts", op="append", T=8100, H=32, Hk=8, d=128, rot=64, ps=64, dtype="fp16",
             interleaved=True, base=10000.0, mscale=1.0, start=0),
        # The smallest call: one request with a short history; latency is all there is.
        dict(name="attend_small", op="attend", B=1, H=16, Hk=4, d=128, length=333, ps=16, dtype="bf16",
             window=0, cap=0.0, slopes=False, lse=False),
        # The ordinary decoding step: a batch of requests of unequal length, grouped heads.
        dict(name="attend_batch", op="attend", B=32, H=32, Hk=8, d=128, length=4096, ps=16, dtype="bf16",
             window=0, cap=0.0, slopes=False, lse=False),
        # One request with a very long history: its keys have to be spread over the GPU.
        dict(name="attend_long", op="attend", B=1, H=32, Hk=8, d=128, length=131072, ps=64, dtype="bf16",
             window=0, cap=0.0, slopes=False, lse=False),
        # A model that caps its scores and looks at a sliding window only, no grouped heads, the smaller head.
        dict(name="attend_capped", op="attend", B=48, H=16, Hk=16, d=64, length=2500, ps=32, dtype="fp16",
             window=1024, cap=30.0, slopes=False, lse=False),
        # A model without rotary positions: a bias by distance; pages of no power of two; and the log-sum-exp,
        # as a caller wants it that joins this with another part of the keys.
        dict(name="attend_bias", op="attend", B=8, H=16, Hk=4, d=128, length=7001, ps=24, dtype="fp16",
             window=0, cap=0.0, slopes=True, lse=True),
        # All query heads on one key head.
        dict(name="attend_shared", op="attend", B=16, H=32, Hk=1, d=128, length=16384, ps=128, dtype="bf16",
             window=0, cap=0.0, slopes=False, lse=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choices(("extend", "rotary", "append", "attend"), (2, 2, 2, 5))[0]
        H = rng.choice((4, 8, 12, 16, 20, 32))
        Hk = H // rng.choice([g for g in (1, 2, 3, 4, 5, 6, 8, 16, 32) if H % g == 0])
        d = rng.choice((64, 128, 128))
        ps = rng.choice((8, 16, 16, 24, 32, 64, 128))
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        turn = dict(rot=rng.choice((d, d, d // 2, d // 4, 20)), interleaved=rng.random() < 0.4,
                    base=rng.choice((10000.0, 500000.0)), mscale=rng.choice((1.0, 1.0, 1.2)),
                    start=rng.choice((0, 0, _log_int(rng, 100, 1000000))))
        if op == "extend":
            one = rng.random() < 0.5
            c = dict(op=op, B=_log_int(rng, 1, 1024), length=_log_int(rng, 1, 8192),
                     new=1 if one else _log_int(rng, 2, 8192), ps=ps)
        elif op == "rotary":
            c = dict(op=op, B=_log_int(rng, 1, 8), S=_log_int(rng, 1, 8192), H=H, Hk=Hk, d=d, dtype=dtype,
                     adjoint=rng.random() < 0.3, **turn)
        elif op == "append":
            c = dict(op=op, T=_log_int(rng, 1, 8192), H=H, Hk=Hk, d=d, ps=ps, dtype=dtype, **turn)
        else:
            c = dict(op=op, B=_log_int(rng, 1, 128), H=H, Hk=Hk, d=d, length=_log_int(rng, 1, 131072), ps=ps,
                     dtype=dtype, window=rng.choice((0, 0, _log_int(rng, 16, 4096))),
                     cap=rng.choice((0.0, 0.0, 30.0, 50.0)), slopes=rng.random() < 0.25, lse=rng.random() < 0.3)
            if 4 * c["B"] * Hk * c["length"] * d > MOST_BYTES[op]:      # the whole history is held, also under a window
                continue
        if work(c)["bytes"] <= MOST_BYTES[op]:
            return c


def _spread(n, most, least):
    """n lengths between least and most, the same for every seed, so that the work of a case is known; the
    first is the longest."""
    return [max(least, int(round(most * (1.0 - 0.7 * ((i * 0.6180339887) % 1.0))))) for i in range(n)]


def _extend_lens(c):
    """(lengths before, new tokens): one request in nine is new, one in eleven is a lane without a token."""
    B = c["B"]
    old = [0 if i % 9 == 4 else n for i, n in enumerate(_spread(B, c["length"], 1))]
    new = [0 if i % 11 == 7 else n for i, n in enumerate(_spread(B, c["new"], 1))]
    return old, new


def _dtype(c):
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float16


def _ceil(a, b):
    return -(-a // b)


def prepare(case, seed):
    c, op = dict(case), case["op"]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def normal(*shape):
        return torch.randn(*shape, device="cuda", dtype=_dtype(c), generator=gen)

    def pages(n):
        """The numbers 1 .. n in an order that the seed gives, as a server's free list ends up."""
        return (torch.randperm(n, device="cuda", generator=gen) + 1).to(torch.int32)

    s = dict(c)
    if "rot" in c:
        i = torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda")
        s["freqs"] = c["base"] ** (-i / c["rot"])
    if op == "extend":
        old, new = _extend_lens(c)
        width = _ceil(c["length"] + c["new"], c["ps"]) + 1
        held = sum(_ceil(n, c["ps"]) for n in old)
        wanted = sum(_ceil(a + n, c["ps"]) - _ceil(a, c["ps"]) for a, n in zip(old, new))
        free = pages(held + wanted + 5)
        col = torch.arange(width, device="cuda")
        have = ints([_ceil(n, c["ps"]) for n in old])
        first = (torch.cumsum(have, 0) - have).unsqueeze(1) + col
        s["table"] = torch.where(col < have.unsqueeze(1), free[first.clamp(max=held + wanted)], -1).to(torch.int32)
        s["free"], s["head"] = free, ints([held])
        s["lens"], s["new"], s["T"] = ints(old), ints(new), sum(new) + 3      # three rows of padding
    elif op == "rotary":
        s["q"] = normal(c["B"], c["S"], c["H"], c["d"]).transpose(1, 2)
        s["k"] = normal(c["B"], c["S"], c["Hk"], c["d"]).transpose(1, 2)
        s["positions"] = ints(range(c["S"])) + c["start"] + 7 * ints(range(c["B"])).unsqueeze(1)
    elif op == "append":
        T, H, Hk, d, ps = c["T"], c["H"], c["Hk"], c["d"], c["ps"]
        n = _ceil(T, ps) + 4
        qkv = normal(T, (H + 2 * Hk) * d)                                # as one projection leaves them
        s["q"] = qkv[:, :H * d].view(T, H, d)
        s["k"], s["v"] = (qkv[:, (H + i * Hk) * d:(H + (i + 1) * Hk) * d].view(T, Hk, d) for i in (0, 1))
        s["positions"] = ints(range(T)) % 2039 + c["start"]
        at = torch.arange(T, device="cuda")
        slots = pages(n - 1)[at // ps].long() * ps + at % ps
        s["slots"] = torch.where(at % 97 == 96, -1, slots)               # rows of padding
        s["k_cache"], s["v_cache"] = normal(n, Hk, ps, d), normal(n, Hk, ps, d)
    else:
        lens = _spread(c["B"], c["length"], 1)
        held = [_ceil(n, c["ps"]) for n in lens]
        width = max(held) + 2
        col = torch.arange(width, device="cuda")
        have = ints(held)
        first = (torch.cumsum(have, 0) - have).unsqueeze(1) + col
        order = pages(sum(held))
        s["table"] = torch.where(col < have.unsqueeze(1), order[first.clamp(max=sum(held) - 1)], 0).to(torch.int32)
        s["lens"] = ints(lens)
        s["q"] = normal(c["B"], c["H"], c["d"])
        s["k_cache"] = normal(1 + sum(held), c["Hk"], c["ps"], c["d"])
        s["v_cache"] = normal(1 + sum(held), c["Hk"], c["ps"], c["d"])
        if c["slopes"]:
            s["slope"] = 2.0 ** (-8.0 * torch.arange(1, c["H"] + 1, dtype=torch.float32, device="cuda") / c["H"])
    return s


# ------------------------------------------------------------------ the plain forms
def _extend(s):
    ps, width = s["ps"], s["table"].shape[1]
    lens, new, free = s["lens"].long(), s["new"].long().clamp(min=0), s["free"]
    old = (lens + ps - 1) // ps
    after = (lens + new + ps - 1) // ps
    fits = after <= width
    need = torch.where(fits, after - old, 0)
    upto = torch.cumsum(need, 0)
    head = s["head"].long()
    granted = fits & ((need == 0) | (upto <= free.numel() - head))
    taken = torch.where(granted, need, 0)
    col = torch.arange(width, device=lens.device)
    source = (head + (upto - need).unsqueeze(1) + col - old.unsqueeze(1)).clamp(0, free.numel() - 1)
    fresh = granted.unsqueeze(1) & (col >= old.unsqueeze(1)) & (col < after.unsqueeze(1))
    s["table"].copy_(torch.where(fresh, free[source], s["table"]))
    cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    t = torch.arange(s["T"], device=lens.device)
    b = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=lens.numel() - 1)
    inside = t < cu[-1]
    pos = torch.where(inside, lens[b] + t - cu[b], 0)
    page = s["table"][b, (pos // ps).clamp(max=width - 1)].long()
    slots = torch.where(inside & granted[b], page * ps + pos % ps, -1)
    return (s["table"], torch.where(granted, lens + new, lens).int(), (head + taken.sum()).int(), slots, pos.int(),
            cu.int())


def _turn(x, angle, s, sign=1.0):
    """x (..., heads, d), angle (..., 1, rot / 2) in 64 bits: the first `rot` elements turned, in 32 bits."""
    cos, sin = (angle.cos() * s["mscale"]).float(), (angle.sin() * (s["mscale"] * sign)).float()
    x = x.float()
    if s["interleaved"]:
        a, b = x[..., 0:s["rot"]:2], x[..., 1:s["rot"]:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :s["rot"] // 2], x[..., s["rot"] // 2:s["rot"]]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([y, x[..., s["rot"]:]], dim=-1)


def _rotary(s):
    angle = (s["positions"].double().unsqueeze(-1) * s["freqs"]).unsqueeze(1)
    sign = -1.0 if s["adjoint"] else 1.0
    return [_turn(s[n], angle, s, sign).to(s[n].dtype).contiguous() for n in ("q", "k")]


def _append(s):
    angle = (s["positions"].double().unsqueeze(-1) * s["freqs"]).unsqueeze(1)
    q, k = (_turn(s[n], angle, s).to(s[n].dtype) for n in ("q", "k"))
    slot, kept = s["slots"].clamp(min=0), (s["slots"] >= 0).view(-1, 1, 1)
    page, row = slot // s["ps"], slot % s["ps"]
    for cache, x in ((s["k_cache"], k), (s["v_cache"], s["v"])):
        cache[page, :, row] = torch.where(kept, x, cache[page, :, row])    # padding rewrites page 0 with itself
    return q, s["k_cache"], s["v_cache"]


def _attend(s):
    B, H, d = s["q"].shape
    Hk, ps = s["k_cache"].shape[1:3]
    q = s["q"].float().view(B, Hk, H // Hk, d)
    k, v = (s[n][s["table"].long()].transpose(1, 2).reshape(B, Hk, -1, d).float() for n in ("k_cache", "v_cache"))
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    if s["cap"] > 0:
        x = s["cap"] * torch.tanh(x / s["cap"])
    back = torch.arange(k.shape[2], device=k.device) - (s["lens"].view(B, 1, 1, 1) - 1)      # 0 at the new token
    if s["slopes"]:
        x = x + s["slope"].view(1, Hk, H // Hk, 1) * back
    hidden = back > 0
    if s["window"] > 0:
        hidden = hidden | (back <= -s["window"])
    x = x.masked_fill(hidden, float("-inf"))
    top = x.amax(dim=-1, keepdim=True)
    p = (x - top).exp()
    total = p.sum(dim=-1, keepdim=True)
    out = ((p @ v) / total).view(B, H, d).to(s["q"].dtype)
    if s["lse"]:
        return out, (top + total.log()).view(B, H)
    return out


def run(state):
    s, op = state, state["op"]
    if not own:
        return {"extend": _extend, "rotary": _rotary, "append": _append, "attend": _attend}[op](s)
    from custom_ops_b200 import ops
    if op == "extend":
        return (s["table"],) + tuple(ops.paged_extend(s["table"], s["lens"], s["new"], s["free"], s["head"],
                                                      s["ps"], s["T"]))
    if op == "rotary":
        return list(ops.rotary(s["q"], s["k"], s["positions"], s["freqs"], interleaved=s["interleaved"],
                               mscale=s["mscale"], adjoint=s["adjoint"]))
    if op == "append":
        q = ops.rotary_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_cache"], s["v_cache"],
                              s["freqs"], interleaved=s["interleaved"], mscale=s["mscale"])
        return q, s["k_cache"], s["v_cache"]
    call = ops.paged_attention_lse if s["lse"] else ops.paged_attention
    return call(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], window=s["window"], softcap=s["cap"],
                slopes=s["slope"] if s["slopes"] else None)


# ------------------------------------------------------------------ what the calls cannot do without
def work(case):
    c, op = case, case["op"]
    if op == "extend":
        old, new = _extend_lens(c)
        wanted = sum(_ceil(a + n, c["ps"]) - _ceil(a, c["ps"]) for a, n in zip(old, new))
        return {"bytes": 8.0 * wanted + 12.0 * (sum(new) + 3) + 16.0 * c["B"], "flops": 0.0}
    if op == "rotary":
        rows = c["B"] * c["S"] * (c["H"] + c["Hk"])
        return {"bytes": 4.0 * rows * c["d"] + 4.0 * c["B"] * c["S"] + 4.0 * c["rot"], "flops": 3.0 * rows * c["rot"]}
    if op == "append":
        T, H, Hk = c["T"], c["H"], c["Hk"]
        return {"bytes": 4.0 * T * (H + 2 * Hk) * c["d"] + 12.0 * T + 4.0 * c["rot"],
                "flops": 3.0 * T * (H + Hk) * c["rot"]}
    lens = _spread(c["B"], c["length"], 1)
    keys = [min(n, c["window"]) if c["window"] > 0 else n for n in lens]
    nbytes = 4.0 * sum(keys) * c["Hk"] * c["d"] + 4.0 * c["B"] * c["H"] * c["d"]
    nbytes += 4.0 * sum(_ceil(n, c["ps"]) for n in keys) + 4.0 * c["B"] + (4.0 * c["B"] * c["H"] if c["lse"] else 0.0)
    return {"bytes": nbytes, "flops": 4.0 * c["H"] * c["d"] * sum(keys)}


# ------------------------------------------------------------------ in 64 bits, one request or head at a time
def _exact_turn(x, positions, freqs, c, adjoint=False):
    """x (tokens, heads, d): every pair as a complex number, times mscale * e^(i angle)."""
    x = x.double()
    angle = torch.outer(positions.double(), freqs)
    w = torch.polar(torch.full_like(angle, c["mscale"]), -angle if adjoint else angle).unsqueeze(1)
    r = c["rot"]
    at = torch.arange(r, device=x.device)
    first, second = (at[0::2], at[1::2]) if c["interleaved"] else (at[:r // 2], at[r // 2:])
    z = torch.complex(x[..., first], x[..., second]) * w
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_extend(s):
    table, lens, new, free, ps = s["table"].tolist(), s["lens"].tolist(), s["new"].tolist(), s["free"].tolist(), s["ps"]
    head, left = s["head"].tolist()[0], True
    slots, positions, cu, after = [], [], [0], []
    for row, n, m in zip(table, lens, new):
        want = list(range(_ceil(n, ps), _ceil(n + m, ps)))
        fits = _ceil(n + m, ps) <= len(row)
        if fits and want:
            left = left and head + len(want) <= len(free)
        ok = fits and (left or not want)
        if ok:
            for at in want:
                row[at], head = free[head], head + 1
        slots += [row[p // ps] * ps + p % ps if ok else -1 for p in range(n, n + m)]
        positions += range(n, n + m)
        cu.append(cu[-1] + m)
        after.append(n + m if ok else n)
    pad = s["T"] - cu[-1]
    out = (table, after, [head], slots + [-1] * pad, positions + [0] * pad, cu)
    return tuple(torch.tensor(x, dtype=torch.int64 if i == 3 else torch.int32, device="cuda") for i, x in enumerate(out))


def exact(case, seed):
    c, op = dict(case), case["op"]
    s = prepare(c, seed)
    if op == "extend":
        return _exact_extend(s)
    if op == "rotary":
        out = []
        for x in (s["q"], s["k"]):
            y = torch.stack([_exact_turn(x[b].transpose(0, 1), s["positions"][b], s["freqs"], c, c["adjoint"])
                             for b in range(c["B"])])
            out.append(y.transpose(1, 2).contiguous())
        return out
    if op == "append":
        q, k = (_exact_turn(s[n], s["positions"], s["freqs"], c) for n in ("q", "k"))
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        kept = s["slots"] >= 0
        slot = s["slots"][kept]
        kc[slot // c["ps"], :, slot % c["ps"]] = k[kept]
        vc[slot // c["ps"], :, slot % c["ps"]] = s["v"][kept].double()
        return q, kc, vc
    B, H, d = s["q"].shape
    out = torch.zeros(B, H, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(B, H, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        lo = max(0, n - c["window"]) if c["window"] > 0 else 0
        key = torch.arange(lo, n, device="cuda")
        page, row = s["table"][b].long()[key // c["ps"]], key % c["ps"]
        for h in range(c["Hk"]):
            k, v = s["k_cache"][page, h, row].double(), s["v_cache"][page, h, row].double()
            heads = slice(h * H // c["Hk"], (h + 1) * H // c["Hk"])
            x = s["q"][b, heads].double() @ k.T / math.sqrt(d)
            if c["cap"] > 0:
                x = torch.tanh(x / c["cap"]) * c["cap"]
            if c["slopes"]:
                x = x - s["slope"][heads].double().unsqueeze(1) * (n - 1 - key)
            lse[b, heads] = torch.logsumexp(x, dim=-1)
            out[b, heads] = torch.softmax(x, dim=-1) @ v
    return (out, lse) if c["lse"] else out
