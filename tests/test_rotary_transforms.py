"""``rotary`` under torch's transforms: batched gradients, vmap, grad and jvp of
torch.func, forward mode, tracing, views that are negative.  The turn is linear, so
that each of these is the turn, or the turn back, of something.  On the CPU a plain
turn stands in for the kernel."""

import pytest
import torch
import torch.autograd.forward_ad as fwd


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


@pytest.mark.parametrize("strategy", ["reverse-mode", "forward-mode"])
def test_jacobian(device, turn, strategy):
    x = heads(device)
    got = torch.autograd.functional.jacobian(turn[0], x, vectorize=True, strategy=strategy)
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


def test_func_grad(device, turn):
    x, y = heads(device), heads(device, seed=1)
    assert torch.equal(torch.func.grad(lambda v: (turn[0](v) * y).sum())(x), turn[1](y))
    out, pull = torch.func.vjp(turn[0], x)
    assert torch.equal(out, turn[0](x)) and torch.equal(pull(y)[0], turn[1](y))


def test_func_grad_of_a_batch(device, turn):
    xs, ys = heads(device, 3), heads(device, 3, seed=1)
    got = torch.func.vmap(torch.func.grad(lambda v, y: (turn[0](v) * y).sum()))(xs, ys)
    assert torch.equal(got, each(turn[1], ys))


def test_func_grad_of_the_gradient(device, turn):
    """Of a square's sum: twice the turn of a turn back, which is factor^2."""
    x, v = heads(device), heads(device, seed=1)
    first = torch.func.grad(lambda u: (turn[0](u) ** 2).sum())
    got = torch.func.grad(lambda u: (first(u) * v).sum())(x)
    assert torch.equal(got, turn[1](2 * turn[0](v)))


def test_jvp(device, turn):
    x, t = heads(device), heads(device, seed=1)
    out, tangent = torch.func.jvp(turn[0], (x,), (t,))
    assert torch.equal(out, turn[0](x)) and torch.equal(tangent, turn[0](t))
    got = torch.func.jacfwd(turn[0])(x)
    assert torch.equal(got, torch.func.jacrev(turn[0])(x).to(got.dtype))


def test_jvp_of_the_gradient(device, turn):
    """Forward over reverse: of half a square's sum, along t."""
    x, t = heads(device), heads(device, seed=1)
    _, got = torch.func.jvp(torch.func.grad(lambda u: 0.5 * (turn[0](u) ** 2).sum()), (x,), (t,))
    assert torch.equal(got, turn[1](turn[0](t)))


def test_forward_mode(device, turn):
    x, t = heads(device), heads(device, seed=1)
    for leaf in (x, x.clone().requires_grad_()):
        with fwd.dual_level():
            out, tangent = fwd.unpack_dual(turn[0](fwd.make_dual(leaf, t)))
            assert torch.equal(out, turn[0](x)) and torch.equal(tangent, turn[0](t))
            assert fwd.unpack_dual(turn[0](leaf)).tangent is None
        assert out.requires_grad == leaf.requires_grad


def test_a_leaf_beside_the_transform(device, turn):
    """What a transform does not see keeps its own gradient."""
    leaf, v, y = heads(device).requires_grad_(), heads(device, seed=1), heads(device, seed=2)
    got = torch.func.grad(lambda u: (turn[0](leaf) * u).sum())(v)
    assert torch.equal(got, turn[0](leaf.detach()))
    assert torch.equal(torch.autograd.grad(got, leaf, y)[0], turn[1](y))


def test_hessian(device, turn):
    """Of half a square's sum: the turn's product with its transpose."""
    x = heads(device)[:1]
    op, pos, freqs = torch.ops.quantized_ops.rotary, turn[2][2:3], turn[3]
    f = lambda u: 0.5 * (op(u, pos, freqs, factor=2.0) ** 2).sum()  # noqa: E731
    want = torch.ones(2, 16, device=device)
    want[:, :12] = 4.0  # factor^2 where heads are turned
    # two turns, each rounded once, and the pair's sum: of terms up to 4
    for got in (torch.func.hessian(f)(x), torch.func.jacrev(torch.func.jacrev(f))(x)):
        assert float((got.reshape(32, 32) - torch.diag(want.flatten())).abs().max()) <= 4 * 2.0 ** -23


def test_tangents_and_gradients_together(device, turn):
    """Forward over reverse and reverse over forward, without torch.func."""
    x, t, y = heads(device).requires_grad_(), heads(device, seed=1), heads(device, seed=2)
    with fwd.dual_level():
        out, tangent = fwd.unpack_dual(turn[0](fwd.make_dual(x, t) ** 2))
        got, = torch.autograd.grad(tangent, x, y)  # of the turn of 2 x t
        assert torch.equal(got, turn[1](y) * 2 * t) or torch.equal(got, turn[1](y) * (2 * t))
        dual = fwd.make_dual(x, t)
        first, = torch.autograd.grad(turn[0](dual).square().sum(), dual, create_graph=True)
        assert torch.equal(fwd.unpack_dual(first).tangent, turn[1](2 * turn[0](t)))


def test_tangents_of_frequencies_are_refused(device, turn):
    x = heads(device)
    with fwd.dual_level(), pytest.raises(ValueError, match="freqs have no gradient"):
        torch.ops.quantized_ops.rotary(x, turn[2], fwd.make_dual(turn[3], turn[3]))


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


def test_frequencies_that_are_a_parameter(device, turn):
    """Are refused where a gradient of them could be asked for, and only there."""
    op, x, freqs = torch.ops.quantized_ops.rotary, heads(device), torch.nn.Parameter(turn[3])
    with torch.no_grad():
        for leaf in (x, x.clone().requires_grad_()):
            assert torch.equal(op(leaf, turn[2], freqs), op(x, turn[2], turn[3]))
    for leaf in (x, x.clone().requires_grad_()):
        with pytest.raises(ValueError, match="freqs have no gradient"):
            op(leaf, turn[2], freqs)
    leaf = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(op(leaf, turn[2], freqs.detach()).sum(), leaf)[0],
                       op(torch.ones_like(x), turn[2], turn[3], back=True))
