"""Scores of the paged attention held to bounds that follow each key's own score and weight, not the largest of the
call: capped scores with caps of any size, and biases by distance of which far keys have thousands."""
import math

import pytest
import torch

from custom_ops_b200 import ops
from tests.paged_testlib import make_cache

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16)


# ------------------------------------------------------------------ the capped score by itself
@pytest.mark.parametrize("cap", [1e-3, 5.0, 30.0, 64.0, 65.0, 1e3, 1e4, 1e6, 1e8, 1e20, 2e38])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,H,Hk,B", [(64, 8, 1, 70), (128, 8, 1, 70), (64, 16, 1, 35), (128, 16, 1, 35), (64, 32, 1, 18),
                                      (128, 32, 1, 18), (64, 4, 2, 500), (128, 4, 2, 500)])
def test_capped_score_of_a_single_key(cap, dtype, d, H, Hk, B):
    """A request with one key has the key's score as its log-sum-exp.  Query and key have one element that is not
    zero, so q.k is exact.  What the cap adds is no more than three approximate steps of 2^-22 times a cap of 64, or
    2^-18.9 of the score (the same steps from a quarter of the cap on, where tanh is 0.245).  The way to powers of
    two and back (factor, product, reference, exp2, log2, factor) takes a few 2^-24 of the score and of the reference's
    distance of at most 2^3."""
    x = torch.logspace(-4, 4.75, B * H, dtype=torch.float64)
    x = (x * torch.where(torch.arange(B * H) % 3 == 0, -1.0, 1.0)).to(dtype)
    q = torch.zeros(B, H, d, dtype=dtype, device="cuda")
    q[:, :, 5] = x.view(B, H).cuda()
    k = torch.zeros(2, Hk, 16, d, dtype=dtype, device="cuda")
    k[..., 5] = 1.0
    v = torch.ones_like(k)
    table = torch.ones(B, 1, dtype=torch.int32, device="cuda")
    lens = torch.ones(B, dtype=torch.int32, device="cuda")
    out, lse = ops.paged_attention_lse(q, k, v, table, lens, scale=1.0, softcap=cap)
    want = cap * torch.tanh(q[:, :, 5].double() / cap)
    bound = min(cap, 64.0) * 2.0 ** -21 + 2.0 ** -18.9 * want.abs() + 2.0 ** -21 * (want.abs() + 8.0)
    off = (lse.double() - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()
    assert (out == 1).all()


# ------------------------------------------------------------------ whole calls, key by key
def bounded_reference(q, k_cache, v_cache, table, lens, scale=None, window=0, softcap=0.0, slopes=None):
    """(out, lse, bounds of both) in 64 bits.  Score of key j, in fp32: a sum of d products, off by (d + 10) 2^-24 of the
    sum of their absolute values; a cap as above; the changes of unit, the bias (one rounded slope, one fma), the
    subtraction of a reference that is at most 14 powers of two away, each 2^-22 of what it handles; exp2 2^-22.  Together
    e_j, so that weight j is off by a factor of at most exp(e_j), and the output by sum_j w_j (exp(e_j) - 1)
    (|v_j| + |out|).  A weight enters the product as two 16-bit numbers (2^-18 in bf16; the tests beside this allow
    2^-16 + 2^-18), where fp16 loses what is below 2^-25 of a largest weight of at least 2^6.  n / 8 + 40 additions of 2^-23."""
    B, H, d = q.shape
    P, Hk, ps, _ = k_cache.shape
    G = H // Hk
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    half = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps / 2
    out = torch.zeros(B, H, d, dtype=torch.float64, device=q.device)
    lse = torch.full((B, H), float("-inf"), dtype=torch.float64, device=q.device)
    out_bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    for b, n in enumerate(lens.tolist()):
        lo = max(0, n - window) if window > 0 else 0
        if n <= lo:
            continue
        key = torch.arange(lo, n, device=q.device)
        page = table[b].long()[key // ps]
        for h in range(Hk):
            k, v = k_cache[page, h, key % ps].double(), v_cache[page, h, key % ps].double()
            heads = slice(h * G, (h + 1) * G)
            x = q[b, heads].double() @ k.T * scale
            e = (d + 10) * 2.0 ** -24 * (q[b, heads].double().abs() @ k.abs().T * scale) + 2.0 ** -22 * x.abs()
            if softcap > 0:
                x = softcap * torch.tanh(x / softcap)
                e = e + min(softcap, 64.0) * 2.0 ** -21 + 2.0 ** -18.9 * x.abs()
            if slopes is not None:
                bias = slopes[heads].double().unsqueeze(1) * (key - (n - 1))
                x = x + bias
                e = e + 2.0 ** -22 * (bias.abs() + x.abs())
            top = x.amax(dim=-1, keepdim=True)
            e = e + 2.0 ** -22 * (x.abs() + (x - top).abs() + 15.0)
            w = torch.softmax(x, dim=-1)
            lse[b, heads] = torch.logsumexp(x, dim=-1)
            out[b, heads] = w @ v
            # (a weight that is off by a factor of e^2 and still below 2^-60 of the largest changes nothing; the others
            # are off by little)
            wide = torch.expm1(e.clamp(max=2.0)) * torch.where(x - top < -50.0, torch.zeros_like(w), w)
            assert (e[x - top >= -50.0] < 0.1).all()
            total = wide.sum(dim=-1, keepdim=True)
            more = (key.numel() / 8 + 40) * 2.0 ** -23
            out_bound[b, heads] = (half * 1.01 * out[b, heads].abs() + 1.1 * (wide @ v.abs() + total * out[b, heads].abs())
                                   + (2.0 ** -16 + 2.0 ** -18 + more) * (w @ v.abs()) + tiny
                                   + key.numel() * 2.0 ** -31 * v.abs().amax())
            lse_bound[b, heads] = 1.1 * total.squeeze(1) + more + 2.0 ** -22 * (1.0 + lse[b, heads].abs())
    return out, lse, out_bound, lse_bound


def check(args, what="", **score):
    want, want_lse, bound, lse_bound = bounded_reference(*args, **score)
    out, lse = ops.paged_attention_lse(*args, **score)
    off = (out.double() - want).abs()
    assert (off <= bound).all(), (what, (off / bound).nan_to_num().max().item())
    empty = torch.isneginf(want_lse)
    assert torch.equal(torch.isneginf(lse), empty), what
    off = (lse.double() - want_lse)[~empty].abs()
    assert (off <= lse_bound[~empty]).all(), (what, (off / lse_bound[~empty]).max().item())


def usual_slopes(H):
    return (2.0 ** (-8.0 * torch.arange(1, H + 1) / H)).float().cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,H,Hk", [(128, 12, 4), (64, 12, 1), (128, 32, 1), (64, 8, 8)])
@pytest.mark.parametrize("window", [0, 65, 200])
def test_biased_scores_key_by_key(dtype, d, H, Hk, window):
    args = make_cache([1, 64, 130, 1500, 0, 4099], H=H, Hk=Hk, d=d, page_size=24, dtype=dtype, gen=torch.Generator().manual_seed(3))
    check(args, "usual", window=window, slopes=usual_slopes(H), scale=0.11)
    check(args, "usual, capped", window=window, slopes=usual_slopes(H), scale=0.11, softcap=5.0)
    mixed = usual_slopes(H)                              # some heads without a bias, one towards the oldest key
    mixed[::3], mixed[1] = 0.0, -0.01
    check(args, "mixed", window=window, slopes=mixed, scale=0.11)


@pytest.mark.parametrize("dtype", DTYPES)
def test_steep_biases_key_by_key(dtype):
    args = make_cache([700, 1, 90, 20000], H=4, Hk=2, d=64, page_size=16, dtype=dtype, gen=torch.Generator().manual_seed(8))
    for slope in (100.0, 1.0, 0.05):
        check(args, f"slope {slope}", slopes=torch.full((4,), slope, device="cuda"))
    args = make_cache([700, 1, 90, 300], H=4, Hk=2, d=64, page_size=16, dtype=dtype, gen=torch.Generator().manual_seed(8))
    for slope in (-5.0, -0.2):                           # towards the oldest key, whose bias is the largest number
        check(args, f"slope {slope}", slopes=torch.full((4,), slope, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,H,Hk", [(128, 8, 2), (64, 16, 1), (64, 32, 1)])
@pytest.mark.parametrize("cap", [20.0, 64.0, 80.0, 1e3, 1e4, 1e6, 1e7, 1e30])
def test_capped_scores_key_by_key(dtype, d, H, Hk, cap):
    args = make_cache([1, 90, 700, 2100], H=H, Hk=Hk, d=d, page_size=16, dtype=dtype, gen=torch.Generator().manual_seed(4))
    check(args, "unit scores", softcap=cap)
    check(args, "large scores", softcap=cap, scale=1.0)
    check(args, "biased, a window", softcap=cap, slopes=usual_slopes(H), window=333)


def test_many_short_requests_key_by_key():
    lens = [(0, 1, 17, 30, 9)[b % 5] for b in range(200)]
    args = make_cache(lens, H=16, Hk=4, d=128, page_size=16, dtype=torch.bfloat16, gen=torch.Generator().manual_seed(5))
    check(args, "plain")
    check(args, "all of it", softcap=1e6, slopes=usual_slopes(16), window=11)
