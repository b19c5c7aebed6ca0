"""Paged key/value cache operators on the GPU against plain 64-bit implementations, at the sizes, masks, layouts
and lengths where they can go wrong."""
import math
import random

import pytest
import torch

from custom_ops_b200 import PagedCache, _cabi_paged, ops, rotary_frequencies
from tests.paged_testlib import (attention_reference, check_attention, check_turned, extend_reference, make_cache,
                                 turn_reference)

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def attend_and_check(q, k, v, table, lens, what="", **score):
    want, want_lse, error = attention_reference(q, k, v, table, lens, **score)
    got, lse = ops.paged_attention_lse(q, k, v, table, lens, **score)
    finite = v[torch.isfinite(v.float())]
    check_attention(got, want, error, finite.float().abs().max().item() if finite.numel() else 0.0, what, lse, want_lse)
    assert torch.equal(ops.paged_attention(q, k, v, table, lens, **score), got), what
    return got


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page_size", [1, 7, 16, 24, 64, 256])
def test_attention_lengths_and_page_sizes(dtype, d, page_size):
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 700, page_size, page_size + 1, 0]
    args = make_cache(lens, H=6, Hk=2, d=d, page_size=page_size, dtype=dtype, gen=gen(page_size))
    got = attend_and_check(*args)
    assert (got[0] == 0).all() and (got[-1] == 0).all()


@pytest.mark.parametrize("H,Hk", [(1, 1), (2, 1), (3, 1), (5, 5), (8, 1), (9, 1), (16, 2), (32, 2), (17, 1), (40, 1), (66, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_head_layouts(H, Hk, d):
    args = make_cache([333, 0, 1, 2100, 64], H=H, Hk=Hk, d=d, page_size=16, dtype=DTYPES[H % 2], gen=gen(H))
    attend_and_check(*args)


@pytest.mark.parametrize("window", [0, 1, 2, 63, 64, 65, 200, 5000, 2 ** 40])
@pytest.mark.parametrize("softcap,biased", [(0.0, False), (20.0, False), (0.0, True), (5.0, True)])
def test_attention_scores(window, softcap, biased):
    H, dtype = 12, DTYPES[int(biased)]
    q, k, v, table, lens = make_cache([1, 64, 130, 1500, 0, 4099], H=H, Hk=4, d=128, page_size=24, dtype=dtype, gen=gen(3))
    slopes = (2.0 ** (-8.0 * torch.arange(1, H + 1) / H)).float().cuda() if biased else None
    attend_and_check(q, k, v, table, lens, window=window, softcap=softcap, slopes=slopes, scale=0.11)


def test_attention_scale_and_large_scores():
    q, k, v, table, lens = make_cache([700, 1, 90], H=4, Hk=2, d=64, page_size=16, dtype=torch.float16, gen=gen(8))
    for scale in (0.0, 0.01, 3.0):                       # all keys alike; flat; one key takes nearly everything
        attend_and_check(q, k, v, table, lens, f"scale {scale}", scale=scale)
    attend_and_check(q * 40, k, v, table, lens, "saturated cap", scale=1.0, softcap=30.0)
    big = torch.full((4,), 100.0, device="cuda")         # a bias that leaves the newest key alone
    attend_and_check(q, k, v, table, lens, "steep bias", slopes=big)
    attend_and_check(q, k, v, table, lens, "bias the other way", slopes=-0.05 * big)


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_never_uses_what_it_must_not_see(fill, d):
    """Behind a length, ahead of a window and on unknown pages the cache may hold anything."""
    lens = [1, 5, 100, 999, 0]
    q, k, v, table, n = make_cache(lens, H=8, Hk=2, d=d, page_size=16, dtype=torch.bfloat16, gen=gen(5), fill=fill)
    attend_and_check(q, k, v, table, n, "behind the length")
    window = 37
    for b, length in enumerate(lens):
        for j in range(max(0, length - window)):
            page = table[b, j // 16]
            k[page, :, j % 16] = fill
            v[page, :, j % 16] = fill
    attend_and_check(q, k, v, table, n, "ahead of the window", window=window)


def test_attention_hides_pages_outside_the_cache():
    q, k, v, table, lens = make_cache([100, 333, 40], H=4, Hk=2, d=128, page_size=16, dtype=torch.float16, gen=gen(6))
    table[0, 2], table[1, 0], table[1, 5] = -1, k.shape[0], -2 ** 31
    table[2] = -1                                        # a request with no known page at all
    got = attend_and_check(q, k, v, table, lens)
    assert (got[2] == 0).all()


def test_attention_lengths_are_clamped_to_the_table():
    q, k, v, table, lens = make_cache([64, 30], H=4, Hk=2, d=64, page_size=16, dtype=torch.float16, gen=gen(7), width=4)
    want = ops.paged_attention(q, k, v, table, torch.tensor([64, 0], dtype=torch.int32, device="cuda"))
    got = ops.paged_attention(q, k, v, table, torch.tensor([10 ** 9, -5], dtype=torch.int32, device="cuda"))
    assert torch.equal(got, want)
    out, lse = ops.paged_attention_lse(q, k, v, table[:, :0], lens)     # a table without columns
    assert (out == 0).all() and torch.isneginf(lse).all()
    assert ops.paged_attention(q[:0], k, v, table[:0], lens[:0]).shape == (0, 4, 64)


@pytest.mark.parametrize("d", [64, 128])
def test_attention_layouts_and_strides(d):
    q, k, v, table, lens = make_cache([70, 500, 3], H=8, Hk=2, d=d, page_size=16, dtype=torch.bfloat16, gen=gen(9))
    want = ops.paged_attention(q, k, v, table, lens)
    by_token = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]          # (P, page_size, Hk, d)
    assert torch.equal(ops.paged_attention(q, *by_token, table, lens), want)
    both = torch.stack([k, v], dim=1)                                                    # one buffer for both
    assert torch.equal(ops.paged_attention(q, both[:, 0], both[:, 1], table, lens), want)
    assert torch.equal(ops.paged_attention(q, k, both[:, 1], table, lens), want)          # different strides
    wide = torch.zeros(3, 5, 8, d, dtype=q.dtype, device="cuda")
    wide[:, 2] = q
    assert torch.equal(ops.paged_attention(wide[:, 2], k, v, table, lens), want)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.paged_attention(heads_first, k, v, table, lens), want)
    cut = torch.zeros(3, table.shape[1] + 9, dtype=torch.int32, device="cuda")[:, 4:4 + table.shape[1]]
    cut.copy_(table)
    assert torch.equal(ops.paged_attention(q, k, v, cut, lens), want)
    row = q[1:2].expand(3, -1, -1)                                                       # one row for all requests
    assert torch.equal(ops.paged_attention(row, k, v, table, lens), ops.paged_attention(row.contiguous(), k, v, table, lens))


def test_attention_offsets_beyond_32_bits():
    """Pages whose first element lies more than 2^31 elements into the cache, by page and by head stride."""
    ps, Hk, d = 16, 2, 128
    P = (2 ** 31 + 2 ** 20) // (Hk * ps * d)
    k = torch.empty(P, Hk, ps, d, dtype=torch.bfloat16, device="cuda")
    pages = [0, P - 1, P - 2, 5, P - 7]
    for p in pages:
        k[p] = torch.randn(Hk, ps, d, device="cuda", generator=torch.Generator("cuda").manual_seed(p))
    table = torch.tensor([pages], dtype=torch.int32, device="cuda")
    lens = torch.tensor([77], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, d, device="cuda").bfloat16()
    small = k[pages].clone()
    want = ops.paged_attention(q, small, small, torch.arange(5, dtype=torch.int32, device="cuda").view(1, 5), lens)
    assert torch.equal(ops.paged_attention(q, k, k, table, lens), want)
    by_head = k.view(Hk, P, ps, d).transpose(0, 1)
    rows = small.transpose(1, 2).reshape(-1, Hk, d)                      # written by the append, token by token
    slots = torch.cat([torch.arange(p * ps, (p + 1) * ps) for p in pages]).cuda()
    by_head_v = torch.empty_like(k).view(Hk, P, ps, d).transpose(0, 1)
    ops.paged_append(rows, rows, slots, by_head, by_head_v)
    for p in pages:
        assert torch.equal(by_head[p], small[pages.index(p)]) and torch.equal(by_head_v[p], by_head[p])
    assert torch.equal(ops.paged_attention(q, by_head, by_head, table, lens), want)


@pytest.mark.parametrize("B,H,Hk,d,length", [(1, 8, 1, 128, 70001), (1, 32, 8, 128, 20000), (2, 4, 4, 64, 33333),
                                             (37, 8, 4, 128, 900), (300, 4, 2, 64, 65), (1500, 2, 1, 64, 20),
                                             (200, 8, 4, 128, 700), (160, 6, 3, 64, 2500), (60, 40, 5, 128, 1200),
                                             (40, 32, 1, 128, 5000), (33, 12, 1, 64, 4000)])
def test_attention_split_over_the_gpu(B, H, Hk, d, length):
    """Long and many: shares begin and end anywhere.  The same call gives the same bits."""
    r = random.Random(B)
    lens = [length] + [r.randint(0, length) for _ in range(B - 1)]
    args = make_cache(lens, H=H, Hk=Hk, d=d, page_size=16, dtype=torch.bfloat16, gen=gen(B))
    got = attend_and_check(*args)
    for _ in range(3):
        assert torch.equal(ops.paged_attention(*args), got)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("H,Hk,B", [(16, 16, 28), (32, 32, 17), (40, 5, 120), (6, 2, 300), (21, 7, 75)])
def test_attention_of_many_short_requests(d, H, Hk, B):
    """More units than CTAs: one warp each, or shares with many ends of units."""
    r = random.Random(B)
    slopes = (2.0 ** (-8.0 * torch.arange(1, H + 1) / H)).float().cuda()
    for most in (1, 20, 350):
        lens = [r.choice((0, 1, 17, most, r.randint(0, most))) for _ in range(B)]
        args = make_cache(lens, H=H, Hk=Hk, d=d, page_size=24, dtype=DTYPES[most % 2], gen=gen(most), fill=float("nan"))
        attend_and_check(*args, what=f"up to {most}")
        attend_and_check(*args, what=f"up to {most}, all of it", window=19, softcap=20.0, slopes=slopes)
    args = make_cache([1000 if b % 9 == 0 else 130 for b in range(B)], H=H, Hk=Hk, d=d, page_size=64, dtype=torch.float16, gen=gen(B))
    attend_and_check(*args, what="a window", window=100)


@pytest.mark.parametrize("d,H,Hk", [(128, 8, 2), (64, 4, 4), (128, 32, 1)])
def test_attention_of_one_long_among_many_short(d, H, Hk):
    """Shares that hold hundreds of ends of units, and a unit that is cut in most of the parts."""
    for B in (5, 31, 32, 33, 150, 700):
        lens = [(0, 1, 70)[b % 3] for b in range(B)]
        lens[B // 2] = 30000
        args = make_cache(lens, H=H, Hk=Hk, d=d, page_size=64, dtype=torch.bfloat16, gen=gen(B))
        attend_and_check(*args, what=f"{B} requests")


@pytest.mark.parametrize("d,H,Hk", [(128, 8, 2), (64, 3, 3), (128, 32, 1), (64, 24, 2)])
def test_attention_of_few_short_requests(d, H, Hk):
    """Few units of few tiles, whatever the table could hold: every way of dividing them up."""
    tile = 8192 // d
    for columns in (1, 2, 3, 5, 8, 9, 17, 33, 64, 65):
        for B in (1, 3, 20):
            r = random.Random(columns + B)
            lens = [columns * tile] + [r.choice((0, 1, r.randint(0, columns * tile))) for _ in range(B - 1)]
            args = make_cache(lens, H=H, Hk=Hk, d=d, page_size=tile, dtype=torch.bfloat16, gen=gen(columns), width=columns)
            attend_and_check(*args, what=f"{columns} columns, {B} requests")
            attend_and_check(*args, what=f"{columns} columns, {B} requests", window=tile + 3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_many_small_weights(dtype):
    """One key takes most; each of 60000 others has a weight of 2^-25.4 of it, below fp16's smallest number, and
    together they are three roundings of the output."""
    n, d = 60001, 64
    q, k, v, table, lens = make_cache([n], H=4, Hk=1, d=d, page_size=16, dtype=dtype, gen=gen(9))
    q.zero_()
    q[..., 0] = 1.0
    k.zero_()
    key = 12345
    k[table[0, key // 16].long(), :, key % 16, 0] = 17.6 if dtype == torch.float16 else 17.625
    v.abs_()
    attend_and_check(q, k, v, table, lens, scale=1.0)


def test_attention_over_a_cache_without_pages():
    q, k, v, table, lens = make_cache([30, 0], H=4, Hk=2, d=128, page_size=16, dtype=torch.float16, gen=gen(1))
    out, lse = ops.paged_attention_lse(q, k[:0], v[:0], table, lens)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_operators_through_compile():
    """As the framework's other operators: traced by their fake kernels, mutations of the caches included."""
    q, k, v, table, lens = make_cache([30, 1, 99], H=4, Hk=2, d=64, page_size=16, dtype=torch.bfloat16, gen=gen(3))
    freqs, _ = rotary_frequencies(64, 10000.0)
    new = torch.randn(3, 8, 64, device="cuda").bfloat16()

    def step(q, new, kc, vc, table, lens, free, head):
        one = torch.ones_like(lens)
        lens, head, slots, positions, _ = ops.paged_extend(table, lens, one, free, head, 16, 3)
        q = ops.rotary_append(new[:, :4], new[:, 4:6], new[:, 6:], positions, slots, kc, vc, freqs)
        return ops.paged_attention(q, kc, vc, table, lens, softcap=20.0), lens, slots

    ops.ensure_loaded("paged")
    got = []
    for f in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        state = [x.clone() for x in (k, v, table, lens)]
        free, head = torch.tensor([k.shape[0] - 1, k.shape[0] - 2], dtype=torch.int32, device="cuda"), torch.zeros_like(lens[:1])
        got.append([*f(q, new, *state, free, head), *state])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_attention_passes_nan_on():
    """A NaN that a row may see is its result, in every way of dividing the work up; other rows are untouched."""
    for length in (40, 700, 9000):
        q, k, v, table, lens = make_cache([length, 50], H=4, Hk=2, d=64, page_size=16, dtype=torch.float16, gen=gen(1))
        want = ops.paged_attention(q, k, v, table, lens)
        q[0, 1, 5] = float("nan")
        out, lse = ops.paged_attention_lse(q, k, v, table, lens)
        assert out[0, 1].isnan().all() and lse[0, 1].isnan()
        keep = torch.ones(2, 4, dtype=torch.bool)
        keep[0, 1] = False
        assert torch.equal(out[keep.cuda()], want[keep.cuda()])


def test_attention_of_each_request_alone():
    """A request's result does not depend on its neighbours beyond where its keys are cut."""
    q, k, v, table, lens = make_cache([2000, 17, 640, 0, 333], H=8, Hk=2, d=128, page_size=16, dtype=torch.float16, gen=gen(2))
    got = ops.paged_attention(q, k, v, table, lens)
    for b in range(5):
        one = ops.paged_attention(q[b:b + 1], k, v, table[b:b + 1], lens[b:b + 1])
        # two roundings of two fp32 results: a step of fp16 and the join's fp32 rounding
        assert ((one[0].float() - got[b].float()).abs() <= 2.0 ** -10 * got[b].float().abs() + 1e-5).all()


def test_attention_in_graphs_and_on_streams():
    """Two captured graphs and an eager call, replayed side by side with new lengths."""
    sets = [make_cache([900, 30, 4000], H=8, Hk=2, d=128, page_size=16, dtype=torch.bfloat16, gen=gen(s)) for s in (1, 2)]
    for s in sets:
        ops.paged_attention(*s)
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in sets], [], []
    for s, stream in zip(sets, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(ops.paged_attention(*s))
        graphs.append(g)
    for step in (0, 1, 7):
        for s in sets:
            s[4].copy_(torch.tensor([900 - step, 30 - step, 4000 - 100 * step], dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(5):
            for g, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    g.replay()
        torch.cuda.synchronize()
        for s, out in zip(sets, outs):
            assert torch.equal(out, ops.paged_attention(*s))


def test_attention_refusals():
    q, k, v, table, lens = make_cache([20, 3], H=4, Hk=2, d=64, page_size=8, dtype=torch.float16, gen=gen(1))
    bad = [
        (dict(q=q.float()), "float16 or bfloat16"), (dict(q=q.bfloat16()), "dtype must match"), (dict(q=q[0]), "3D"),
        (dict(q=q[:, :3]), "divisible"), (dict(k=k[0]), "4D"), (dict(v=v[:, :1]), "one shape"), (dict(v=v.bfloat16()), "match"),
        (dict(k=k[..., ::2], v=v[..., ::2]), "head_dim"), (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
        (dict(q=torch.zeros(2 * 4 * 64 + 1, device="cuda").half()[1:].view(2, 4, 64)), "aligned"),
        (dict(q=torch.zeros(2, 4, 68, device="cuda").half()[..., :64]), "multiples of 8"),
        (dict(table=table.long()), "int32"), (dict(table=table[:1]), "one row per request"), (dict(table=table[0]), "2D"),
        (dict(table=table.t().contiguous().t()), "rows of block_table"), (dict(lens=lens.long()), "int32"),
        (dict(lens=lens[:1]), "2 values"), (dict(lens=torch.zeros(4, dtype=torch.int32, device="cuda")[::2]), "contiguous"),
        (dict(lens=lens.cpu()), "CUDA"), (dict(window=-1), "window"), (dict(softcap=-1.0), "softcap"),
        (dict(softcap=float("nan")), "softcap"), (dict(scale=float("inf")), "scale"), (dict(scale=-1.0), "scale"),
        (dict(slopes=torch.ones(3, device="cuda")), "slopes"), (dict(slopes=torch.ones(4, device="cuda").double()), "slopes"),
    ]
    for kw, match in bad:
        a = dict(q=q, k=k, v=v, table=table, lens=lens)
        score = {n: kw[n] for n in kw if n not in a}
        a.update({n: kw[n] for n in kw if n in a})
        with pytest.raises(RuntimeError, match=match):
            ops.paged_attention(a["q"], a["k"], a["v"], a["table"], a["lens"], **score)


# ------------------------------------------------------------------ tables
def random_tables(seed):
    g = random.Random(seed)
    B, W, ps, F = g.choice((1, 2, 9, 40)), g.randint(0, 7), g.choice((1, 3, 8, 16)), g.randint(0, 60)
    lens = [g.randint(-2, W * ps) for _ in range(B)]
    new = [g.choice((0, 0, 1, 1, g.randint(-1, 3 * ps + 1))) for _ in range(B)]
    T = max(0, sum(max(n, 0) for n in new) + g.choice((0, 0, 5, -2)))
    i32 = dict(dtype=torch.int32)
    table = torch.arange(B * W, **i32).view(B, W) + 1000
    free = torch.randperm(F, generator=gen(seed)).to(torch.int32) + 1
    return table, torch.tensor(lens, **i32), torch.tensor(new, **i32), free, torch.tensor([g.randint(0, F)], **i32), ps, T


def check_extend(table, lens, new, free, head, ps, T):
    want = extend_reference(table, lens, new, free, head, ps, T)
    dev = [x.cuda() for x in (table, lens, new, free, head)]
    got = (dev[0],) + tuple(ops.paged_extend(*dev, ps, T))
    for name, x, y in zip(("table", "lens", "head", "slots", "positions", "cu"), got, want):
        if name == "lens":
            y = [max(v, 0) for v in y]
        assert x.tolist() == y, name
    assert dev[1].tolist() == lens.tolist() and dev[4].tolist() == head.tolist()
    dev = [x.cuda() for x in (table, lens, new, free, head)]
    slots, positions, cu = ops.paged_extend_(*dev, ps, T)
    for x, y in zip((dev[0], dev[1], dev[4], slots, positions, cu), got):
        assert x.tolist() == y.tolist()
    return dev, got


@pytest.mark.parametrize("seed", range(24))
def test_extend_against_the_plain_loop(seed):
    check_extend(*random_tables(seed))


@pytest.mark.parametrize("B,W,ps,most,F", [(1, 400, 16, 6000, 500), (1025, 12, 16, 150, 9000), (3000, 6, 8, 40, 7000),
                                           (64, 40, 128, 5000, 2000), (16384, 2, 4, 7, 20000)])
def test_extend_many(B, W, ps, most, F):
    r = random.Random(B)
    i32 = dict(dtype=torch.int32)
    lens = torch.tensor([r.randint(0, most) for _ in range(B)], **i32)
    new = torch.tensor([r.choice((0, 1, r.randint(0, max(0, W * ps - n)))) for n in lens.tolist()], **i32)
    table = torch.randint(0, F, (B, W), generator=gen(1), **i32)
    free = torch.randperm(F, generator=gen(2)).to(torch.int32)
    check_extend(table, lens, new, free, torch.tensor([3], **i32), ps, int(new.sum()) + 7)


def test_extend_edges():
    i32 = dict(dtype=torch.int32)
    none, one = torch.zeros(0, **i32), torch.zeros(1, **i32)
    check_extend(torch.zeros(0, 4, **i32), none, none, none, one, 16, 3)                 # no request, only padding
    check_extend(torch.zeros(1, 0, **i32), one, one + 5, one, one, 16, 5)                # a table without columns
    check_extend(torch.zeros(2, 3, **i32), torch.tensor([48, 47], **i32), torch.tensor([1, 1], **i32), one, one, 16, 2)
    head = torch.tensor([9], **i32)                                                      # a head behind the list
    dev = [x.cuda() for x in (torch.zeros(1, 2, **i32), one, one + 1, one, head)]
    lens, after, slots, _, _ = ops.paged_extend(*dev, 4, 1)
    assert lens.tolist() == [0] and slots.tolist() == [-1] and after.tolist() == [1]
    # rows of a wider table, and what lies beside them
    wide = torch.full((3, 10), -7, **i32, device="cuda")
    ops.paged_extend(wide[:, 2:6], *[x.cuda() for x in (one.expand(3).contiguous(), one.expand(3).contiguous() + 17,
                                                        torch.arange(50, **i32), one)], 8, 51)
    assert wide[:, 2:5].flatten().tolist() == list(range(9)) and (wide[:, 5:] == -7).all() and (wide[:, :2] == -7).all()


@pytest.mark.parametrize("seed", range(12))
def test_shrink_gives_back_what_extend_gave(seed):
    r = random.Random(seed)
    B, W, ps, F = r.choice((1, 5, 33, 1100)), 9, r.choice((1, 4, 16)), 12000
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens, head = torch.zeros(B, W, **i32), torch.zeros(B, **i32), torch.zeros(1, **i32)
    free = torch.randperm(F, generator=gen(seed)).to(torch.int32).cuda()
    whole = sorted(free.tolist())
    for _ in range(4):
        new = torch.tensor([r.randint(0, 3 * ps) for _ in range(B)], **i32)
        ops.paged_extend_(table, lens, new, free, head, ps, 1)
        keep = torch.tensor([r.choice((0, -1, 10 ** 9, r.randint(0, W * ps))) for _ in range(B)], **i32)
        before = lens.tolist()
        ops.paged_shrink_(table, lens, keep, free, head, ps)
        assert lens.tolist() == [max(0, min(a, b)) for a, b in zip(before, keep.tolist())]
        held = [p for row, n in zip(table.tolist(), lens.tolist()) for p in row[:-(-n // ps)]]
        assert len(held) == head.item() and sorted(held + free.tolist()[head.item():]) == whole
    ops.paged_shrink_(table, lens, torch.zeros(B, **i32), free, head, ps)
    assert head.item() == 0 and sorted(free.tolist()) == whole and not lens.any()


def test_shrink_refuses_pages_that_never_came_from_the_list():
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.arange(6, **i32).view(2, 3)
    lens, free, head = torch.tensor([5, 12], **i32), torch.full((4,), 99, **i32), torch.tensor([2], **i32)
    ops.paged_shrink_(table, lens, torch.zeros(2, **i32), free, head, 4)
    assert lens.tolist() == [0, 12] and head.item() == 0 and free.tolist() == [0, 1, 99, 99]


def test_table_refusals():
    i32 = dict(dtype=torch.int32, device="cuda")
    t, n, f, h = torch.zeros(3, 4, **i32), torch.zeros(3, **i32), torch.arange(9, **i32), torch.zeros(1, **i32)
    for args, match in (((t.long(), n, n, f, h, 8, 3), "int32"), ((t[0], n, n, f, h, 8, 3), "2D"), ((t, n[:2], n, f, h, 8, 3), "3 values"),
                        ((t, n, n.long(), f, h, 8, 3), "int32"), ((t, n, n, f[::2], h, 8, 3), "contiguous"),
                        ((t, n, n, f, n, 8, 3), "1 values"), ((t, n, n, f, h, 0, 3), "positive"), ((t, n, n, f, h, 8, -1), "num_tokens"),
                        ((t, n, n, f, h, 2 ** 30, 3), "32 bits"), ((t.t().contiguous().t(), n, n, f, h, 8, 3), "rows"),
                        ((t[:1].expand(3, 4), n, n, f, h, 8, 3), "overlap|single memory"), ((t, n, n, f, h.cpu(), 8, 3), "CUDA")):
        with pytest.raises(RuntimeError, match=match):
            ops.paged_extend(*args)
    big = torch.zeros(16385, **i32)
    with pytest.raises(RuntimeError, match="16384"):
        ops.paged_extend(torch.zeros(16385, 1, **i32), big, big, f, h, 8, 1)


# ------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rot", [2, 16, 20, 32, 62, 64, 128])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_against_the_formula(dtype, d, rot, interleaved):
    if rot > d:
        pytest.skip("rot_dim above head_dim is refused")
    g = gen(rot)
    B, H, Hk, S = 2, 5, 3, 37
    q = torch.randn(B, S, H, d, generator=g).to(dtype).cuda().transpose(1, 2)
    k = torch.randn(B, Hk, S, d, generator=g).to(dtype).cuda()
    freqs, _ = rotary_frequencies(rot, 10000.0)
    positions = torch.randint(0, 2 ** 20, (B, S), generator=g, dtype=torch.int32).cuda()
    for mscale, adjoint in ((1.0, False), (1.37, True)):
        got = ops.rotary(q, k, positions, freqs, interleaved, mscale, adjoint)
        for x, y in zip((q, k), got):
            assert y.is_contiguous()
            check_turned(y, turn_reference(x, positions.unsqueeze(1), freqs, interleaved, mscale, adjoint), (mscale, adjoint))
            assert torch.equal(y[..., rot:], x[..., rot:])


def test_rotary_positions_far_and_of_either_kind():
    freqs, _ = rotary_frequencies(128, 500000.0)
    far = [0, 1, -1, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31]
    q = torch.randn(1, 3, len(far), 128, device="cuda").half()
    for dtype in (torch.int32, torch.int64):
        p = torch.tensor(far, dtype=dtype, device="cuda")
        a, b = ops.rotary(q, q[:, :1], p, freqs)
        check_turned(a, turn_reference(q, p, freqs))
        assert torch.equal(b, a[:, :1])
        assert torch.equal(a[:, :, 0], q[:, :, 0])                       # position 0 turns nothing
    # An angle of 2^40 is itself known to 2^40 * 2^-53 = 2^-13 in 64 bits only, in the plain form as here: the
    # product with the frequency is rounded once there; here it is, then the factor 1 / (2 pi) is (2^-54 off)
    # and the product with it: (1 + 1 + 0.5 + 1) * 2^-13 between the two.
    p = torch.tensor([2 ** 40 + 3], dtype=torch.int64, device="cuda")
    a, _ = ops.rotary(q[:, :, :1], q[:, :, :1], p, freqs)
    check_turned(a, turn_reference(q[:, :, :1], p, freqs), angle_error=3.5 * 2.0 ** -13)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_adjoint_is_the_gradient(interleaved):
    """Against autograd through the formula in 64 bits, and against differences of the operator itself."""
    freqs, _ = rotary_frequencies(20, 100.0)
    p = torch.arange(7, dtype=torch.int32, device="cuda") * 3
    x = torch.randn(1, 2, 7, 64, device="cuda").half()
    dy = torch.randn(1, 2, 7, 64, device="cuda").half()
    leaf = x.double().requires_grad_()
    angle = p.double().unsqueeze(-1) * freqs
    at = torch.arange(20, device="cuda")
    first, second = (at[0::2], at[1::2]) if interleaved else (at[:10], at[10:])
    a, b = leaf[..., first], leaf[..., second]
    y = leaf.clone()
    y[..., first] = 1.25 * (a * angle.cos() - b * angle.sin())
    y[..., second] = 1.25 * (b * angle.cos() + a * angle.sin())
    y.backward(dy.double())
    dx, _ = ops.rotary(dy, dy, p, freqs, interleaved, 1.25, adjoint=True)
    check_turned(dx, leaf.grad)
    # the map is linear: a difference along any direction e is exact up to rounding, <dy, F(x + e) - F(x)> = <dx, e>
    for i in (0, 3, 19, 20, 63):
        e = torch.zeros_like(x)
        e[..., i] = 0.5
        up, _ = ops.rotary(x + e, x, p, freqs, interleaved, 1.25)
        down, _ = ops.rotary(x - e, x, p, freqs, interleaved, 1.25)
        step = ((x + e).double() - (x - e).double())
        got = (dy.double() * (up.double() - down.double())).sum(-1)
        want = (leaf.grad * step).sum(-1)
        # up and down are rounded to fp16 (2^-11 of at most 1.25 * 2 * |x|); at most three elements differ
        bound = 2.0 ** -11 * 1.25 * 2 * 2 * 3 * (x.abs().max().item() + 0.5) * dy.abs().max().item()
        assert (got - want).abs().max().item() <= bound


def test_rotary_shapes_and_refusals():
    freqs, _ = rotary_frequencies(64, 10000.0)
    x = torch.randn(2, 3, 5, 64, device="cuda").bfloat16()
    p = torch.arange(5, dtype=torch.int32, device="cuda")
    for q, k in ((x[:0], x[:0]), (x[:, :0], x), (x, x[:, :0]), (x[:, :, :0], x[:, :, :0])):
        a, b = ops.rotary(q, k, p[:q.shape[2]], freqs)
        assert a.shape == q.shape and b.shape == k.shape
    both, _ = ops.rotary(x, x, p.expand(2, 5), freqs)                    # one row of positions for the batch
    assert torch.equal(both, ops.rotary(x, x, p, freqs)[0])
    one, _ = ops.rotary(x[:1].expand(2, -1, -1, -1), x, p, freqs)
    assert torch.equal(one[1], both[0])
    bad = ((x.float(), x, p, freqs), (x, x.half(), p, freqs), (x[0], x, p, freqs), (x, x[:1], p, freqs), (x, x, p[:4], freqs),
           (x, x, p.float(), freqs), (x, x, p, freqs.float()), (x, x, p, freqs[:0]), (x, x, p, torch.cat([freqs, freqs])),
           (x, x, p, freqs[::2]), (x[..., :32], x[..., :32], p, freqs[:8]), (x, x, p.cpu(), freqs),
           (x.transpose(2, 3).contiguous().transpose(2, 3), x, p, freqs), (x, x, p.view(1, 1, 5), freqs))
    for args in bad:
        with pytest.raises(RuntimeError):
            ops.rotary(*args)
    with pytest.raises(RuntimeError):
        ops.rotary(x, x, p, freqs, mscale=float("nan"))


def test_rotary_offsets_beyond_32_bits():
    """More than 2^31 elements in and out, rows one behind the other and interleaved by head."""
    H, S, d = 33, 2 ** 19 + 3, 128
    q = torch.empty(1, S, H, d, dtype=torch.float16, device="cuda").transpose(1, 2)
    at = torch.tensor([0, 1, S // 2, S - 2, S - 1], device="cuda")
    q[:, :, at] = torch.randn(1, H, 5, d, device="cuda").half()
    freqs, _ = rotary_frequencies(d, 10000.0)
    out, _ = ops.rotary(q, q[:, :0], torch.arange(S, device="cuda"), freqs)
    check_turned(out[:, :, at], turn_reference(q[:, :, at], at, freqs))


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,rot,interleaved", [(64, 64, False), (128, 128, False), (128, 32, True), (64, 20, False)])
@pytest.mark.parametrize("page_size", [1, 16, 24])
def test_append_writes_its_slots_and_nothing_else(dtype, d, rot, interleaved, page_size):
    g, T, H, Hk, P = gen(d + rot), 53, 6, 2, 70
    qkv = torch.randn(T, (H + 2 * Hk) * d, generator=g).to(dtype).cuda()
    q, k, v = qkv[:, :H * d].view(T, H, d), qkv[:, H * d:(H + Hk) * d].view(T, Hk, d), qkv[:, (H + Hk) * d:].view(T, Hk, d)
    kc, vc = [torch.randn(P, Hk, page_size, d, generator=g).to(dtype).cuda() for _ in range(2)]
    slots = torch.randperm(P * page_size, generator=g)[:T].cuda()
    slots[3], slots[11], slots[20], slots[52] = -1, P * page_size, 2 ** 40, -2 ** 50
    positions = torch.randint(0, 5000, (T,), generator=g).cuda()
    freqs, _ = rotary_frequencies(rot, 10000.0)
    for s in (slots, slots.clamp(-2, P * page_size).int()):
        for copy in (False, True):
            kk, vv = (x.transpose(1, 2).contiguous().transpose(1, 2) if copy else x.clone() for x in (kc, vc))
            out = ops.rotary_append(q, k, v, positions if copy else positions.int(), s, kk, vv, freqs, interleaved, 1.1)
            check_turned(out, turn_reference(q, positions.unsqueeze(1), freqs, interleaved, 1.1))
            kept = (slots >= 0) & (slots < P * page_size)
            at = slots[kept]
            check_turned(kk[at // page_size, :, at % page_size],
                         turn_reference(k[kept], positions[kept].unsqueeze(1), freqs, interleaved, 1.1))
            assert torch.equal(vv[at // page_size, :, at % page_size], v[kept])
            rest = torch.ones(P * page_size, dtype=torch.bool, device="cuda")
            rest[at] = False
            for x, y in ((kk, kc), (vv, vc)):
                assert torch.equal(x.transpose(1, 2).reshape(-1, Hk, d)[rest], y.transpose(1, 2).reshape(-1, Hk, d)[rest])
    kk, vv = kc.clone(), vc.clone()
    ops.paged_append(k, v, slots, kk, vv)
    assert torch.equal(kk[at // page_size, :, at % page_size], k[kept]) and torch.equal(vv[at // page_size, :, at % page_size], v[kept])


def test_append_the_same_slot_twice_leaves_rows_of_the_two():
    x = torch.stack([torch.full((2, 64), 1.0), torch.full((2, 64), 2.0)]).half().cuda()
    c = torch.zeros(2, 2, 2, 2, 4, 64, dtype=torch.float16, device="cuda")
    ops.paged_append(x, x, torch.tensor([5, 5], device="cuda"), c[0, 0], c[1, 0])
    row = c[:, 0, 1, :, 1]
    assert ((row == 1) | (row == 2)).all() and c.count_nonzero() == row.numel()


def test_append_refusals():
    x, c = torch.zeros(3, 2, 64, device="cuda").half(), torch.zeros(4, 2, 8, 64, device="cuda").half()
    c2, s, p = c.clone(), torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    freqs, _ = rotary_frequencies(64, 10000.0)
    for args in ((x.float(), x, s, c, c2), (x, x.bfloat16(), s, c, c2), (x[:2], x, s, c, c2), (x[:, :1], x[:, :1], s, c, c2),
                 (x, x, s[:2], c, c2), (x, x, s.float(), c, c2), (x, x, s, c, c2[:3]), (x, x, s, c, c), (x, x, s.cpu(), c, c2),
                 (x, x, s, c[:1].expand(4, -1, -1, -1), c2), (x[..., :32], x[..., :32], s, c, c2), (x, x, s, c[0], c2[0])):
        with pytest.raises(RuntimeError):
            ops.paged_append(*args)
    for q, pos in ((x[:2], p), (x, p[:2]), (x.bfloat16(), p), (x[0], p), (x, p.float())):
        with pytest.raises(RuntimeError):
            ops.rotary_append(q, x, x, pos, s, c, c2, freqs)
    ops.paged_append(x[:0], x[:0], s[:0], c, c2)


def test_operands_inside_what_is_written_are_refused():
    c, c2 = (torch.zeros(4, 2, 8, 64, device="cuda").half() for _ in range(2))
    x, s = torch.zeros(3, 2, 64, device="cuda").half(), torch.zeros(3, dtype=torch.int64, device="cuda")
    freqs, _ = rotary_frequencies(64, 10000.0)
    for inside in (c.view(-1, 2, 64)[4:7], c2.view(-1, 2, 64)[:3]):
        for k, v in ((inside, x), (x, inside)):
            with pytest.raises(RuntimeError, match="memory location"):
                ops.paged_append(k, v, s, c, c2)
        with pytest.raises(RuntimeError, match="memory location"):
            ops.rotary_append(inside, x, x, s, s, c, c2, freqs)
    lens = torch.full((9,), 5, dtype=torch.int32, device="cuda")
    table, free = torch.zeros(8, 2, dtype=torch.int32, device="cuda"), torch.arange(16, dtype=torch.int32, device="cuda")
    head = torch.full((1,), 16, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="memory location"):
        ops.paged_shrink_(table, lens[:8], lens[1:], free, head, 4)
    ops.paged_shrink_(table, lens[:8], lens[:8], free, head, 4)          # one tensor: nothing changes
    assert (lens == 5).all() and head.item() == 16


# ------------------------------------------------------------------ together
def layered_reference(tokens_q, tokens_k, tokens_v, freqs, mscale, upto):
    """Attention of the token at `upto - 1` of one request over its first `upto` tokens, in 64 bits, from the
    unturned projections; k and v rounded to the cache's type as the cache does."""
    pos = torch.arange(upto, device="cuda")
    q = turn_reference(tokens_q[upto - 1], pos[-1:], freqs, mscale=mscale).to(tokens_q.dtype).double()
    k = turn_reference(tokens_k[:upto], pos.unsqueeze(1), freqs, mscale=mscale).to(tokens_k.dtype).double()
    G = q.shape[0] // k.shape[1]
    x = torch.einsum("hd,jhd->hj", q, k.repeat_interleave(G, dim=1)) / math.sqrt(q.shape[-1])
    return torch.einsum("hj,jhd->hd", torch.softmax(x, dim=-1), tokens_v[:upto].double().repeat_interleave(G, dim=1))


def test_a_decoding_server_end_to_end():
    """Prompts enter a cache of two layers, their attention runs through the masked-attention operator; then
    tokens are decoded one by one by a captured step; requests leave and others take their pages."""
    B, H, Hk, d, layers, dtype = 4, 8, 2, 128, 2, torch.bfloat16
    freqs, mscale = rotary_frequencies(d, 10000.0, scaling="by_parts", factor=4.0, original_length=64)
    cache = PagedCache(layers=layers, num_pages=40, page_size=16, heads_k=Hk, head_dim=d, max_requests=B, max_length=200,
                       dtype=dtype)
    n, steps = [37, 1, 100, 0], 20
    g = gen(77)
    toks = [[[torch.randn(150, h, d, generator=g).to(dtype).cuda() for h in (H, Hk, Hk)] for _ in range(B)] for _ in range(layers)]
    new = torch.tensor(n, dtype=torch.int32, device="cuda")
    T = sum(n) + 6
    slots, positions, cu = cache.extend(new, T)
    assert cache.seq_lens.tolist() == n and cu.tolist() == [0, 37, 38, 138, 138] and (slots[138:] == -1).all()
    for layer in range(layers):
        packed = [torch.cat([toks[layer][b][i][:n[b]] for b in range(B)] + [torch.zeros(6, h, d, dtype=dtype, device="cuda")])
                  for i, h in enumerate((H, Hk, Hk))]
        turned = cache.append(layer, *packed, slots, positions, freqs, mscale=mscale)
        # the prompt's own attention: the same turned queries and keys through the rule operator
        for b in (0, 2):
            q, k, v = [toks[layer][b][i][:n[b]].transpose(0, 1).unsqueeze(0) for i in range(3)]
            qt, kt = ops.rotary(q, k, torch.arange(n[b], device="cuda"), freqs, mscale=mscale)
            assert torch.equal(qt[0].transpose(0, 1), turned[cu[b]:cu[b + 1]])
            prompt = ops.mha_fwd_rule_mask(qt, kt, v.contiguous(), causal=True)
            last = cache.attend(layer, turned[cu[1:].long() - 1])[b]
            want = layered_reference(*toks[layer][b], freqs, mscale, n[b])
            # the rule operator rounds its weights to bf16 (2^-8) and both round the output (2^-8)
            assert (last.double() - want).abs().max() <= 2.0 ** -7 * want.abs().max()
            assert (prompt[0, :, -1].double() - want).abs().max() <= 2.0 ** -6 * want.abs().max()

    one = torch.tensor([1, 1, 1, 0], dtype=torch.int32, device="cuda")
    ins = [[torch.zeros(B, h, d, dtype=dtype, device="cuda") for h in (H, Hk, Hk)] for _ in range(layers)]

    def step():
        slots, positions, _ = cache.extend(one, B)
        outs = []
        for layer in range(layers):
            q = cache.append(layer, *ins[layer], slots, positions, freqs, mscale=mscale)
            outs.append(cache.attend(layer, q))
        return outs

    saved = [x.clone() for x in (cache.seq_lens, cache.free_head, cache.block_table, cache.k, cache.v)]
    step()                                                # a first pass outside the capture, and back
    for x, y in zip((cache.seq_lens, cache.free_head, cache.block_table, cache.k, cache.v), saved):
        x.copy_(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for t in range(steps):
        for layer in range(layers):
            for i in range(3):
                for b in range(3):
                    ins[layer][i][b] = toks[layer][b][i][n[b] + t]
        graph.replay()
        assert cache.seq_lens.tolist() == [n[0] + t + 1, n[1] + t + 1, n[2] + t + 1, 0]
        if t % 7 == 0 or t == steps - 1:
            for layer in range(layers):
                for b in range(3):
                    want = layered_reference(*toks[layer][b], freqs, mscale, n[b] + t + 1)
                    assert (outs[layer][b].double() - want).abs().max() <= 2.0 ** -7 * want.abs().max(), (t, layer, b)
                assert (outs[layer][3] == 0).all()
    held = cache.free_head.item()
    cache.release(torch.tensor([0, 2], device="cuda"))
    assert cache.seq_lens.tolist() == [0, n[1] + steps, 0, 0]
    assert cache.free_head.item() == -(-(n[1] + steps) // 16) and held > cache.free_head.item()
    mine = set(cache.block_table[1, :cache.free_head.item()].tolist())
    cache.extend(torch.tensor([0, 0, 0, 150], dtype=torch.int32, device="cuda"), 150)
    theirs = set(cache.block_table[3, :10].tolist())
    assert cache.seq_lens.tolist()[3] == 150 and not (mine & theirs) and 0 not in theirs


def test_decode_form_agrees_with_the_rule_operator():
    """One query row per request under valid lengths, through both operators."""
    B, H, Hk, d, S = 5, 16, 4, 128, 700
    lens = [1, 64, 333, 700, 0]
    q, k, v, table, n = make_cache(lens, H=H, Hk=Hk, d=d, page_size=16, dtype=torch.float16, gen=gen(12))
    full = [torch.zeros(B, Hk, S, d, dtype=torch.float16, device="cuda") for _ in range(2)]
    for b, length in enumerate(lens):
        j = torch.arange(length, device="cuda")
        for x, c in zip(full, (k, v)):
            x[b, :, :length] = c[table[b].long()[j // 16], :, j % 16].transpose(0, 1)
    want = ops.mha_fwd_rule_mask(q.unsqueeze(2), *full, valid_lens=n).squeeze(2)
    got = ops.paged_attention(q, k, v, table, n)
    # weights rounded to fp16 on one side, one output rounding on each: 3 * 2^-11 of the largest value
    assert (got.float() - want.float()).abs().max().item() <= 3 * 2.0 ** -11 * v.float().abs().max().item()


def test_launches_are_counted():
    q, k, v, table, lens = make_cache([2000], H=8, Hk=2, d=128, page_size=16, dtype=torch.float16, gen=gen(4))
    ops.paged_attention(q, k, v, table, lens)
    before = _cabi_paged.launch_count()
    ops.paged_attention(q, k, v, table, lens)
    assert 1 <= _cabi_paged.launch_count() - before <= 2
