"""Gradients recorded through ``ops.rotary``: their wiring on meta tensors (CPU), their values on the GPU."""
import pytest
import torch

from custom_ops_b200 import ops, rotary_frequencies
from tests.paged_testlib import check_turned, turn_reference

DTYPES = (torch.bfloat16, torch.float16)


# ------------------------------------------------------------------ wiring (CPU)
def meta(*shape, dtype=torch.bfloat16, grad=False):
    return torch.empty(*shape, dtype=dtype, device="meta", requires_grad=grad)


def test_gradients_reach_the_inputs_that_want_them():
    p, f = meta(5, dtype=torch.int32), meta(8, dtype=torch.float64)
    for wants_q, wants_k in ((True, True), (True, False), (False, True)):
        q, k = meta(2, 4, 5, 64, grad=wants_q), meta(2, 1, 5, 64, grad=wants_k)
        a, b = ops.rotary(q, k, p, f, interleaved=True, mscale=1.5)
        assert a.requires_grad and b.requires_grad
        (a.sum() + b.sum()).backward()
        for x, wants in ((q, wants_q), (k, wants_k)):
            assert (x.grad is not None) == wants
            assert not wants or (x.grad.shape == x.shape and x.grad.dtype == x.dtype)


def test_nothing_is_recorded_where_nothing_wants_a_gradient():
    p, f = meta(5, dtype=torch.int32), meta(8, dtype=torch.float64)
    q = meta(2, 4, 5, 64, grad=True)
    assert not any(y.requires_grad for y in ops.rotary(q.detach(), q.detach(), p, f))
    with torch.no_grad():
        assert not any(y.requires_grad for y in ops.rotary(q, q, p, f))
    with torch.inference_mode():
        assert not any(y.requires_grad for y in ops.rotary(q, q, p, f))


def test_frequencies_that_want_a_gradient_are_refused():
    q, p = meta(2, 4, 5, 64), meta(5, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="freqs"):
        ops.rotary(q, q, p, meta(8, dtype=torch.float64, grad=True))
    with torch.no_grad():
        ops.rotary(q, q, p, meta(8, dtype=torch.float64, grad=True))


# ------------------------------------------------------------------ values (GPU)
def inputs(dtype, d, B=2, H=6, Hk=2, S=19, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, S, H, d, generator=g).to(dtype).cuda().transpose(1, 2)
    k = torch.randn(B, Hk, S, d, generator=g).to(dtype).cuda()
    p = torch.randint(0, 10000, (B, S), generator=g, dtype=torch.int32).cuda()
    return q, k, p


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,rot,interleaved", [(64, 64, False), (128, 32, True), (64, 20, False)])
def test_gradient_against_the_formula(dtype, d, rot, interleaved):
    q, k, p = inputs(dtype, d)
    freqs, _ = rotary_frequencies(rot, 10000.0)
    q.requires_grad_(), k.requires_grad_()
    a, b = ops.rotary(q, k, p, freqs, interleaved, 1.25)
    da, db = torch.randn_like(a), torch.randn_like(b)
    gq, gk = torch.autograd.grad((a, b), (q, k), (da, db))
    for got, dy in ((gq, da), (gk, db)):
        check_turned(got, turn_reference(dy, p.unsqueeze(1), freqs, interleaved, 1.25, adjoint=True))
    want = ops.rotary(da, db, p, freqs, interleaved, 1.25, adjoint=True)
    assert torch.equal(gq, want[0]) and torch.equal(gk, want[1])
    # the gradient of the adjoint is the way there
    a, b = ops.rotary(q, k, p, freqs, interleaved, 1.25, adjoint=True)
    gq, _ = torch.autograd.grad((a, b), (q, k), (da, db))
    assert torch.equal(gq, ops.rotary(da, db, p, freqs, interleaved, 1.25)[0])


@pytest.mark.gpu
def test_gradients_of_any_layout_and_of_shared_rows():
    q, k, p = inputs(torch.float16, 64)
    freqs, _ = rotary_frequencies(64, 10000.0)
    q.requires_grad_()
    a, b = ops.rotary(q, k, p, freqs)
    dy = torch.randn_like(a)
    want = ops.rotary(dy, b, p, freqs, adjoint=True)[0]
    # a strided gradient, one that is broadcast, one of a part, and none at all for the other output
    strided = dy.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(torch.autograd.grad(a, q, strided, retain_graph=True)[0], want)
    odd = torch.empty(dy.numel() + 1, dtype=dy.dtype, device="cuda")[1:].view(dy.shape).copy_(dy)
    assert torch.equal(torch.autograd.grad(a, q, odd, retain_graph=True)[0], want)
    ones = torch.autograd.grad(a.sum(), q, retain_graph=True)[0]
    assert torch.equal(ones, ops.rotary(torch.ones_like(a), b, p, freqs, adjoint=True)[0])
    part = torch.autograd.grad((a[:, :, 3:, 32:].float() * dy[:, :, 3:, 32:].float()).sum(), q, retain_graph=True)[0]
    some = torch.zeros_like(dy)
    some[:, :, 3:, 32:] = dy[:, :, 3:, 32:]
    assert torch.equal(part, ops.rotary(some, b, p, freqs, adjoint=True)[0])
    zero = torch.autograd.grad(b.sum() + 0 * a.sum(), q)[0]
    assert not zero.any()
    for part in (q[:, :0], q[:, :, :0], q[:0]):          # and of nothing
        beside = k[:, :, :part.shape[2]] if part.shape[0] else k[:0]
        none, other = ops.rotary(part, beside, p[:part.shape[0], :part.shape[2]], freqs)
        assert not torch.autograd.grad(none.sum() + other.sum(), q)[0].any()
    # one row for the whole batch: its gradient is the sum over the batch, as elsewhere
    row = torch.randn(1, 6, 19, 64, device="cuda").half().requires_grad_()
    a, _ = ops.rotary(row.expand(2, -1, -1, -1), k, p, freqs)
    got = torch.autograd.grad(a, row, dy)[0]
    both = ops.rotary(dy, b, p, freqs, adjoint=True)[0]
    # two fp16 numbers added and rounded once
    assert ((got.double() - both.double().sum(0, keepdim=True)).abs() <= 2.0 ** -11 * 1.01 * got.double().abs() + 2.0 ** -25).all()


@pytest.mark.gpu
def test_second_gradient_and_changed_positions():
    q, k, p = inputs(torch.float16, 64)
    freqs, _ = rotary_frequencies(64, 10000.0)
    q.requires_grad_()
    a, _ = ops.rotary(q, k, p, freqs)
    dy = torch.randn_like(a).requires_grad_()
    g, = torch.autograd.grad(a, q, dy, create_graph=True)
    e = torch.randn_like(g)
    back, = torch.autograd.grad(g, dy, e)                # the map is linear: its gradient's gradient is itself
    assert torch.equal(back, ops.rotary(e, k, p, freqs)[0])
    a, _ = ops.rotary(q, k, p, freqs)
    p.add_(1)                                            # what the gradient needs is gone, and torch says so
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(a.sum(), q)


@pytest.mark.gpu
def test_gradient_through_compile_and_in_a_graph():
    q, k, p = inputs(torch.bfloat16, 128)
    freqs, _ = rotary_frequencies(128, 10000.0)
    dy = torch.randn(q.shape, device="cuda").bfloat16()

    def step(q, k):
        a, b = ops.rotary(q, k, p, freqs, mscale=1.1)
        return (a.float() * dy.float()).sum() + b.float().sum()

    def grads(f):
        x, y = q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_()
        return torch.autograd.grad(f(x, y), (x, y))

    want = grads(step)
    for a, b in zip(want, grads(torch.compile(step, backend="aot_eager", fullgraph=True))):
        assert torch.equal(a, b)
    x, y = q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(step(x, y), (x, y))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = torch.autograd.grad(step(x, y), (x, y))
    for s in (1.0, -2.0):
        with torch.no_grad():
            dy.mul_(s)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, grads(step)):
            assert torch.equal(a, b)
