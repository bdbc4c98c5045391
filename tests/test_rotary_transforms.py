"""``rotary`` under torch's transforms: batched gradients, vmap, tracing, views that
are negative.  The turn is linear, so that each of these is the turn, or the turn
back, of something.  On the CPU a plain turn stands in for the kernel."""

import pytest
import torch


def plain_turn(x, positions, freqs, *, interleaved=False, factor=1.0, back=False):
    r = 2 * freqs.shape[0]
    angle = positions.double()[:, None] * freqs.double()
    z = torch.polar(torch.full_like(angle, factor), -angle if back else angle)[:, None]
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y = x.double().clone()
    w = torch.complex(y[..., a], y[..., b]) * z
    y[..., a], y[..., b] = w.real, w.imag
    return y.to(x.dtype)


@pytest.fixture(scope="module", params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def device(request, vqx):
    if request.param == "cuda":
        yield "cuda"
        return
    with torch.library._scoped_library("quantized_ops", "IMPL") as lib:
        lib.impl("rotary", plain_turn, "CPU")
        yield "cpu"


HOW = [dict(interleaved=False, factor=1.0), dict(interleaved=True, factor=1.5)]


@pytest.fixture(params=HOW, ids=["halves", "neighbours"])
def turn(request, vqx, device):
    """(the turn of x, the turn back, positions, frequencies)"""
    pos, freqs = (torch.arange(5).int() * 77).to(device), vqx.ops.rotary_frequencies(12, device=device)
    op = torch.ops.quantized_ops.rotary
    return (lambda x: op(x, pos, freqs, **request.param), lambda x: op(x, pos, freqs, back=True, **request.param), pos, freqs)


def heads(device, *batch, dtype=torch.float32, seed=0):
    return torch.randn(*batch, 5, 2, 16, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def each(f, xs):
    return torch.stack([f(x) for x in xs])


def test_batched_gradients(device, turn):
    x, ys = heads(device).requires_grad_(), heads(device, 3, seed=1)
    got, = torch.autograd.grad(turn[0](x), x, ys, is_grads_batched=True)
    assert torch.equal(got, each(turn[1], ys))


def test_batched_gradients_of_the_gradient(device, turn):
    x, y, vs = heads(device).requires_grad_(), heads(device, seed=1).requires_grad_(), heads(device, 3, seed=2)
    back, = torch.autograd.grad(turn[0](x), x, y, create_graph=True)
    got, = torch.autograd.grad(back, y, vs, is_grads_batched=True)
    assert torch.equal(got, each(turn[0], vs))


def test_jacobian(device, turn):
    x = heads(device)
    got = torch.autograd.functional.jacobian(turn[0], x, vectorize=True)
    units = torch.eye(x.numel(), device=device).reshape(-1, *x.shape)
    assert torch.equal(got.flatten(3).movedim(-1, 0), each(turn[0], units))


def test_vmap(device, turn):
    xs = heads(device, 4)
    assert torch.equal(torch.func.vmap(turn[0])(xs), each(turn[0], xs))


def test_vmap_of_positions(device, turn):
    op, x, many = torch.ops.quantized_ops.rotary, heads(device), torch.stack([turn[2], turn[2] + 9, -turn[2]])
    got = torch.func.vmap(lambda p: op(x, p, turn[3]))(many)
    assert torch.equal(got, each(lambda p: op(x, p, turn[3]), many))
    leaf = x.clone().requires_grad_()
    got = torch.func.vmap(lambda p: op(leaf, p, turn[3]))(many)
    assert torch.equal(got, each(lambda p: op(x, p, turn[3]), many))


@pytest.mark.parametrize("grad", [False, True])
def test_negative_views(device, turn, grad):
    """The imaginary part of a conjugate is a view that is negative."""
    z = torch.complex(heads(device), heads(device, seed=1)).requires_grad_(grad)
    x = z.conj().imag
    assert x.is_neg()
    assert torch.equal(turn[0](x), turn[0](-z.detach().imag.contiguous()))
    dense = torch._neg_view(z.detach().imag.contiguous()).requires_grad_(grad)
    assert dense.is_neg() and dense.is_contiguous()
    assert torch.equal(turn[0](dense), turn[0](-z.detach().imag.contiguous()))


def test_negative_gradients(device, turn):
    x, y = heads(device).requires_grad_(), heads(device, seed=1)
    got, = torch.autograd.grad(turn[0](x), x, torch._neg_view(y))
    assert torch.equal(got, turn[1](-y))


@pytest.mark.parametrize("grad", [False, True])
def test_compiled_graphs(device, turn, grad):
    """Through the tracer's own kinds of tensors."""
    from torch.fx.experimental.proxy_tensor import make_fx

    op, x = torch.ops.quantized_ops.rotary, heads(device).requires_grad_(grad)

    def both(x, positions, freqs):
        out = op(x, positions, freqs)
        return (out, *torch.autograd.grad(out, x, torch.ones_like(out))) if grad else (out,)

    made = make_fx(both, tracing_mode="fake")(x, *turn[2:])
    assert sum("rotary" in str(n.target) for n in made.graph.nodes) == 1 + grad
    for a, b in zip(made(x, *turn[2:]), both(x, *turn[2:])):
        assert torch.equal(a, b)
