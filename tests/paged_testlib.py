"""Plain 64-bit implementations of the paged-cache operators, and the error bounds their results are held to."""
from __future__ import annotations

import math

import torch


def extend_reference(table, lens, new, free, head, page_size, num_tokens):
    """Python integers throughout: one request after the other."""
    table, lens, new, free, head = [x.tolist() for x in (table, lens, new, free, head)]
    head, left = min(max(head[0], 0), len(free)), True
    after, slots, positions, cu = [], [], [], [0]
    for row, n, m in zip(table, lens, new):
        n, m = max(n, 0), max(m, 0)
        have, want = -(-n // page_size), -(-(n + m) // page_size)
        ok = want <= len(row)
        if ok and want > have:
            left = left and head + want - have <= len(free)
            ok = left
        if ok:
            row[have:want] = free[head:head + want - have]
            head += want - have
        slots += [row[p // page_size] * page_size + p % page_size if ok else -1 for p in range(n, n + m)]
        positions += range(n, n + m)
        cu.append(cu[-1] + m)
        after.append(n + m if ok else n)
    slots = (slots + [-1] * num_tokens)[:num_tokens]
    positions = (positions + [0] * num_tokens)[:num_tokens]
    return table, after, [head], slots, positions, cu


def turn_reference(x, positions, freqs, interleaved=False, mscale=1.0, adjoint=False):
    """x (..., d) in 64 bits, positions broadcastable to x's leading dimensions."""
    x = x.double().clone()
    angle = positions.double().unsqueeze(-1) * freqs.double()
    cos, sin = angle.cos() * mscale, angle.sin() * mscale * (-1.0 if adjoint else 1.0)
    n = freqs.numel()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first].clone(), x[..., second].clone()
    x[..., first] = a * cos - b * sin
    x[..., second] = b * cos + a * sin
    return x


def check_turned(got, want, what="", angle_error=0.0):
    """Angles of positions up to 2^28 are good to better than fp32 (``angle_error``: for others); cos and sin are rounded to fp32 (2^-24, and the scaling by
    mscale once more), two products and a sum in fp32: at most 2^-21 of |a| + |b|.  Then one rounding: half a
    step of the type, relative, or half its smallest subnormal."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    bound = half * 1.01 * want.abs() + 2.0 ** -21 * want.abs().amax(dim=-1, keepdim=True) * 2 + tiny
    bound = bound + angle_error * 2 * want.abs().amax(dim=-1, keepdim=True)
    assert got.shape == want.shape
    off = (got.double() - want).abs() - bound
    assert (off <= 0).all(), (what, off.max().item())


def attention_reference(q, k_cache, v_cache, table, lens, scale=None, window=0, softcap=0.0, slopes=None):
    """(out, lse, bound of |score error|) in 64 bits, one request and key head at a time."""
    B, H, d = q.shape
    P, Hk, ps, _ = k_cache.shape
    G = H // Hk
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(B, H, d, dtype=torch.float64, device=q.device)
    lse = torch.full((B, H), float("-inf"), dtype=torch.float64, device=q.device)
    worst = 0.0
    for b, n in enumerate(lens.tolist()):
        n = min(max(n, 0), table.shape[1] * ps)
        lo = max(0, n - window) if window > 0 else 0
        key = torch.arange(lo, n, device=q.device)
        page = table[b].long()[key // ps] if n > lo else key
        known = (page >= 0) & (page < P)
        key, page = key[known], page[known]
        if key.numel() == 0:
            continue
        for h in range(Hk):
            k = k_cache[page, h, key % ps].double()
            v = v_cache[page, h, key % ps].double()
            heads = slice(h * G, (h + 1) * G)
            x = q[b, heads].double() @ k.T * scale
            worst = max(worst, (q[b, heads].double().abs() @ k.abs().T).max().item() * scale)
            if softcap > 0:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x + slopes[heads].double().unsqueeze(1) * (key - (n - 1))
                worst = max(worst, x.abs().max().item())
            lse[b, heads] = torch.logsumexp(x, dim=-1)
            out[b, heads] = torch.softmax(x, dim=-1) @ v
    return out, lse, score_error(d, worst, softcap)


def score_error(d, worst, softcap):
    """fp32: a sum of d products is off by at most (d + 2) 2^-24 of the sum of their absolute values; the scale,
    the change to powers of two, the bias and the subtraction of the maximum add a few 2^-24 of the score's size,
    exp2 2^-22.  The capped form adds the absolute error of 1 - 2 / (1 + e^2y), three approximate steps of 2^-22
    each, times the cap."""
    return (d + 10) * 2.0 ** -24 * worst + 2.0 ** -22 + softcap * 2.0 ** -21


def check_attention(got, want, error, v_most, what="", lse=None, want_lse=None):
    """A weight is off by a factor of at most e^(2 error) (its score and the sum's); as the sum of two 16-bit
    numbers by 2^-16 (bf16) more; the output is a mean of values of at most v_most.  Then one rounding."""
    assert got.shape == want.shape, what
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    bound = half * 1.01 * want.abs() + v_most * (2.2 * error + 2.0 ** -16 + 2.0 ** -18) + tiny
    off = (got.double() - want).abs() - bound
    assert (off <= 0).all(), (what, off.max().item(), error)
    if lse is not None:
        empty = torch.isneginf(want_lse)
        assert torch.equal(torch.isneginf(lse), empty), what
        err = (lse.double() - want_lse)[~empty].abs()
        assert (err <= error + 2.0 ** -22 * (1.0 + want_lse[~empty].abs())).all(), (what, err.max().item(), error)


def make_cache(lens, *, H, Hk, d, page_size, dtype, gen, extra_pages=3, fill=None, width=None, device="cuda"):
    """q, caches, table for requests of these lengths; pages in random order, page 0 unused.  ``fill``: what the
    cache holds where no token of a request is (else random values)."""
    held = [-(-max(n, 0) // page_size) for n in lens]
    W = max(held + [1]) + 1 if width is None else width
    P = sum(held) + 1 + extra_pages
    order = (torch.randperm(P - 1, generator=gen) + 1).tolist()
    table = torch.full((len(lens), W), 2 ** 31 - 1, dtype=torch.int32)          # never to be looked up
    shape = (P, Hk, page_size, d)
    k, v = (torch.randn(shape, generator=gen).to(dtype) for _ in range(2))
    if fill is not None:
        used = torch.zeros(P, page_size, dtype=torch.bool)
    for b, n in enumerate(lens):
        pages = [order.pop() for _ in range(held[b])]
        table[b, :held[b]] = torch.tensor(pages, dtype=torch.int32)
        if fill is not None:
            for j in range(n):
                used[pages[j // page_size], j % page_size] = True
    if fill is not None:
        for x in (k, v):
            x.masked_fill_(~used[:, None, :, None], fill)
    q = torch.randn(len(lens), H, d, generator=gen).to(dtype)
    return (q.to(device), k.to(device), v.to(device), table.to(device),
            torch.tensor(lens, dtype=torch.int32, device=device))
