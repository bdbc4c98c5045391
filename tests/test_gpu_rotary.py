"""Rotary positions on the GPU: against complex products in 64 bits, as a
gradient, and on the way into the 4-bit cache."""

import math

import pytest
import torch

from tests.test_gpu_kv4 import make_cache, near, on, same

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops(vqx):
    return torch.ops.quantized_ops


def turned(x, positions, freqs, interleaved=False, factor=1.0, back=False):
    """x [n, heads, D] in 64 bits times factor exp(i angle)."""
    r = 2 * freqs.shape[0]
    y = x.double().clone()
    angle = positions.double()[:, None] * freqs.double()
    z = torch.polar(torch.full_like(angle, factor), -angle if back else angle)[:, None]
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    w = torch.complex(y[..., a], y[..., b]) * z
    y[..., a], y[..., b] = w.real, w.imag
    return y


def tolerance(x, want, dtype):
    """The one rounding, to fp32 and on to the type, and 64 bits' own error on
    pairs that cancel."""
    tol = (torch.finfo(dtype).eps / 2 + 2.0 ** -24) * want.abs() + 2.0 ** -48 * x.double().abs().amax(-1, keepdim=True)
    return tol + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -149)


def positions_of(n, far, gen):
    p = torch.randint(0, far, (n,), generator=gen).int()
    p[:1] = 0
    p[-1:] = far - 1
    return p


CASES = [
    # kind, tokens, heads, dim, turned, interleaved, how far, factor
    ("bf16", 1, 1, 8, 2, False, 10, 1.0),
    ("f32", 1, 1, 8, 8, True, 10, 1.0),
    ("bf16", 5, 3, 64, 64, False, 5000, 1.0),
    ("f16", 33, 12, 64, 64, True, 5000, 1.0),
    ("f32", 7, 5, 128, 128, False, 1 << 20, 1.0),
    ("bf16", 257, 32, 128, 128, False, 131073, 1.0),
    ("f16", 100, 8, 256, 64, True, 4000, 0.5),
    ("f32", 31, 2, 256, 256, False, 2 ** 31 - 1, 1.25),
    ("bf16", 19, 3, 64, 24, False, 900, 1.0),  # halves of 12: paired one by one
    ("f16", 19, 3, 72, 24, True, 900, 1.0),
    ("f32", 6, 2, 96, 10, False, 900, -2.0),
    ("bf16", 6, 2, 80, 10, True, 900, 1.0),
    ("bf16", 3, 1, 1024, 1024, False, 900, 1.0),
    ("f32", 2100, 1, 64, 32, False, 2100, 1.0),  # many tokens of one small head
]


@pytest.mark.parametrize("kind,n,heads,dim,r,interleaved,far,factor", CASES)
@pytest.mark.parametrize("back", [False, True])
def test_rotary(ops, vqx, kind, n, heads, dim, r, interleaved, far, factor, back):
    g = torch.Generator().manual_seed(n + dim)
    x = torch.randn(n, heads, dim, generator=g).to(TYPES[kind])
    pos, freqs = positions_of(n, far, g), vqx.ops.rotary_frequencies(r)
    got = ops.rotary(*on(x, pos, freqs), interleaved=interleaved, factor=factor, back=back)
    want = turned(x, pos, freqs, interleaved, factor, back)
    assert got.dtype == x.dtype
    near(got, want, tolerance(x, want, x.dtype) * max(1.0, abs(factor)), "turned")
    same(got[..., r:], x[..., r:], "the rest of the head")


def test_rotary_negative_positions(ops, vqx):
    x, pos, freqs = torch.randn(9, 2, 64), torch.arange(-4, 5).int() * 1000, vqx.ops.rotary_frequencies(64)
    want = turned(x, pos, freqs)
    near(ops.rotary(*on(x, pos, freqs)), want, tolerance(x, want, x.dtype), "turned")


def test_rotary_no_tokens(ops, vqx):
    freqs = vqx.ops.rotary_frequencies(64, device=DEV)
    out = ops.rotary(torch.zeros(0, 3, 64, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV), freqs)
    assert out.shape == (0, 3, 64)
    assert ops.rotary(torch.zeros(4, 0, 64, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV), freqs).shape == (4, 0, 64)


@pytest.mark.parametrize("view", [
    lambda: torch.randn(11, 9, 128).bfloat16().to(DEV)[:, 2:7],          # heads out of a projection
    lambda: torch.randn(5, 11, 128).bfloat16().to(DEV).transpose(0, 1),  # heads before tokens
    lambda: torch.randn(11, 5, 256).bfloat16().to(DEV)[..., 3:131],      # rows off 16 bytes: copied
    lambda: torch.randn(11, 5, 256).bfloat16().to(DEV)[..., ::2],        # elements apart: copied
    lambda: torch.randn(11, 1, 128).bfloat16().to(DEV).expand(11, 5, 128)])
def test_rotary_strides(ops, vqx, view):
    x = view()
    before = x.clone()
    pos, freqs = torch.arange(11).int().to(DEV) * 77, vqx.ops.rotary_frequencies(128, device=DEV)
    got = ops.rotary(x, pos, freqs)
    assert got.is_contiguous() and torch.equal(x, before)
    same(got, ops.rotary(x.contiguous(), pos, freqs).cpu(), "a strided view")


@pytest.mark.parametrize("kind", list(TYPES))
def test_rotary_small_values(ops, vqx, kind):
    """Subnormal values and results are neither lost nor flushed; what is not
    turned comes back bit for bit."""
    tiny = torch.finfo(TYPES[kind]).tiny
    x = (torch.randn(20, 2, 64, dtype=torch.float64, generator=torch.Generator().manual_seed(1)) * tiny).to(TYPES[kind])
    pos, freqs = torch.arange(20).int(), vqx.ops.rotary_frequencies(48)
    for interleaved in (False, True):
        want = turned(x, pos, freqs, interleaved)
        got = ops.rotary(*on(x, pos, freqs), interleaved=interleaved)
        # half a step of the subnormals, once to fp32 and once to the type
        near(got, want, torch.finfo(x.dtype).eps * tiny / 2 + 2.0 ** -149 + torch.finfo(x.dtype).eps / 2 * want.abs(), "turned")
        assert torch.equal(got[..., 48:].cpu().view(torch.uint8), x[..., 48:].contiguous().view(torch.uint8))


def test_rotary_special_values(ops, vqx):
    """What is not finite reaches its own pair only."""
    x = torch.ones(2, 1, 64)
    x[0, 0, 5], x[1, 0, 40] = math.inf, math.nan
    pos, freqs = torch.tensor([0, 3]).int(), vqx.ops.rotary_frequencies(64)
    got = ops.rotary(*on(x, pos, freqs)).cpu()
    bad = torch.zeros(2, 1, 64, dtype=torch.bool)
    bad[0, 0, 5] = bad[0, 0, 37] = bad[1, 0, 40] = bad[1, 0, 8] = True
    assert torch.equal(~got.isfinite(), bad)


@pytest.mark.parametrize("kind,r,interleaved,factor", [("f32", 64, False, 1.0), ("bf16", 64, True, 1.5), ("f16", 20, False, 1.0)])
def test_rotary_gradient(ops, vqx, kind, r, interleaved, factor):
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(13, 3, 64, generator=g).to(TYPES[kind]) for _ in range(2))
    pos, freqs = positions_of(13, 3000, g), vqx.ops.rotary_frequencies(r)
    leaf = x.to(DEV).requires_grad_()
    out = ops.rotary(leaf, *on(pos, freqs), interleaved=interleaved, factor=factor)
    got, = torch.autograd.grad(out, leaf, dy.to(DEV))
    want = turned(dy, pos, freqs, interleaved, factor, back=True)
    near(got, want, tolerance(dy, want, dy.dtype) * factor, "gradient")


def test_rotary_gradient_of_differences(ops, vqx):
    """The map is linear: its gradient along any direction is a difference."""
    g = torch.Generator().manual_seed(4)
    x, d, dy = (torch.randn(6, 2, 32, generator=g).to(DEV) for _ in range(3))
    pos, freqs = torch.arange(6).int().to(DEV) * 50, vqx.ops.rotary_frequencies(32, device=DEV)
    leaf = x.clone().requires_grad_()
    got, = torch.autograd.grad(ops.rotary(leaf, pos, freqs), leaf, dy)
    moved = (ops.rotary(x + d, pos, freqs).double() - ops.rotary(x - d, pos, freqs).double()) / 2
    # roundings of x + d, x - d and of the three results, of values up to 6
    assert abs(float((moved * dy.double()).sum() - (got.double() * d.double()).sum())) < 5 * 6 * 2.0 ** -24 * float(dy.abs().sum())


def test_rotary_gradient_of_a_broadcast_input(ops, vqx):
    """A head that several share gets the sum of their gradients; a second
    derivative is a turn again."""
    pos, freqs = torch.arange(7).int().to(DEV), vqx.ops.rotary_frequencies(64, device=DEV)
    leaf = torch.randn(7, 1, 64, device=DEV, requires_grad=True)
    out = ops.rotary(leaf.expand(7, 4, 64), pos, freqs)
    out.sum().backward()
    want = 4 * turned(torch.ones(7, 1, 64), pos.cpu(), freqs.cpu(), back=True)
    near(leaf.grad, want, 8 * 2.0 ** -24 * (want.abs() + 1), "shared head")
    dy = torch.ones(7, 1, 64, device=DEV, requires_grad=True)
    grad, = torch.autograd.grad(ops.rotary(leaf, pos, freqs), leaf, dy, create_graph=True)
    again, = torch.autograd.grad(grad, dy, torch.ones_like(grad))
    same(again, ops.rotary(torch.ones(7, 1, 64, device=DEV), pos, freqs).cpu(), "second derivative")


def test_rotary_graph(ops, vqx):
    """A captured turn follows positions and values as they change."""
    x = torch.randn(16, 4, 128, device=DEV).bfloat16()
    pos, freqs = torch.zeros(16, dtype=torch.int32, device=DEV), vqx.ops.rotary_frequencies(128, device=DEV)
    ops.rotary(x, pos, freqs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rotary(x, pos, freqs)
    for i in range(4):
        pos.fill_(i * 1234)
        x.copy_(torch.randn(16, 4, 128, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        same(out, ops.rotary(x, pos, freqs).cpu(), f"replay {i}")


def test_rotary_gradient_of_the_gradient(ops, vqx):
    """The turn is linear: the gradient's own gradient is the turn again."""
    x, g, v = (torch.randn(9, 3, 64, device=DEV, requires_grad=True) for _ in range(3))
    pos, freqs = torch.arange(9, device=DEV, dtype=torch.int32) * 77, vqx.ops.rotary_frequencies(48, device=DEV)
    back, = torch.autograd.grad(ops.rotary(x, pos, freqs, factor=1.5), x, g, create_graph=True)
    again, = torch.autograd.grad(back, g, v)
    same(again, ops.rotary(v, pos, freqs, factor=1.5).detach().cpu(), "gradient of the gradient")


def test_rotary_backward_graph(ops, vqx):
    """Forward and backward captured together follow x, positions and gradient."""
    x = torch.randn(16, 4, 128, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = torch.randn(16, 4, 128, device=DEV, dtype=torch.bfloat16)
    pos, freqs = torch.arange(16, device=DEV, dtype=torch.int32), vqx.ops.rotary_frequencies(128, device=DEV)
    call = lambda: torch.autograd.grad(ops.rotary(x, pos, freqs), x, y)[0]  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(4):
        pos.fill_(i * 999)
        y.copy_(torch.randn(16, 4, 128, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        same(got, call().cpu(), f"replay {i}")


# ---------------------------------------------------------------------------
# into the cache
# ---------------------------------------------------------------------------
FUSED = [
    # kind, dim, kv, group, lengths, new, page, turned, interleaved
    ("bf16", 128, 2, 4, [1, 2, 31, 900], 1, 16, 128, False),
    ("f32", 64, 1, 1, [1], 1, 0, 64, True),
    ("f16", 64, 3, 5, [40, 5, 64], None, 24, 24, False),
    ("bf16", 256, 1, 2, [200, 0, 35], None, 0, 64, True),
    ("f32", 128, 8, 1, [130, 77], None, 16, 128, False),
    ("bf16", 64, 4, 8, [2000, 1], None, 256, 32, False),
]


@pytest.mark.parametrize("kind,dim,kv,group,lengths,new,page,r,interleaved", FUSED)
@pytest.mark.parametrize("given", [False, True])
def test_append_rotary_is_rotary_and_append(ops, vqx, kind, dim, kv, group, lengths, new, page, r, interleaved, given):
    """Bit for bit what the calls apart make, in the cache and of the queries."""
    g = torch.Generator().manual_seed(dim + kv)
    seqs = len(lengths)
    news = [new] * seqs if new else [(n * 3 + 3) // 4 for n in lengths]
    total, heads = sum(news), kv * group
    codes, scales, table = make_cache(seqs, kv, dim, max(max(lengths), 1), page, seed=1)
    cu = torch.tensor([0] + news).cumsum(0).int() if not new else None
    qkv = torch.randn(total, heads + 2 * kv, dim, generator=g).to(TYPES[kind]).to(DEV)
    q, k, v = qkv.split([heads, kv, kv], 1)
    lens = torch.tensor(lengths).int()
    places = torch.cat([torch.arange(n - t, n) for n, t in zip(lengths, news)]).int()
    pos = (places + torch.randint(0, 100000, (total,), generator=g).int()) if given else places
    freqs = vqx.ops.rotary_frequencies(r, device=DEV)
    one, two = on(codes, scales), on(codes, scales)
    dl, dcu, dt, dpos = on(lens, cu, table, pos)
    got = ops.kv4_append_rotary(q, k, v, *one, dl, freqs, dcu, dt, dpos if given else None, interleaved=interleaved,
                                factor=1.5)
    want = ops.rotary(q, dpos, freqs, interleaved=interleaved, factor=1.5)
    ops.kv4_append(ops.rotary(k, dpos, freqs, interleaved=interleaved, factor=1.5), v, *two, dl, dcu, dt)
    same(got, want.cpu(), "queries")
    same(one[0], two[0].cpu(), "codes")
    same(one[1], two[1].cpu(), "scales")


def test_append_rotary_rows_behind_the_last_sequence(ops, vqx):
    """Tokens of no sequence are not written; neither are those without a page."""
    codes, scales, table = make_cache(2, 1, 64, 32, 16)
    table[1] = -1
    dev = on(codes, scales, torch.tensor([5, 3]).int(), torch.tensor([0, 2, 3]).int(), table)
    q, k, v = (torch.randn(6, 1, 64, device=DEV) for _ in range(3))
    out = ops.kv4_append_rotary(q, k, v, dev[0], dev[1], dev[2], vqx.ops.rotary_frequencies(64, device=DEV), dev[3], dev[4])
    assert out.shape == (6, 1, 64)
    page, slots = int(table[0, 0]), [3, 4]
    keep = torch.ones(codes.shape[1:4], dtype=torch.bool)
    keep[page, :, slots] = False
    for got, was in ((dev[0], codes), (dev[1], scales)):
        for plane in (0, 1):
            assert torch.equal(got[plane].cpu()[keep], was[plane][keep])
            assert not torch.equal(got[plane].cpu()[~keep], was[plane][~keep])
