"""Sampled tokens against loops over sorted Python lists, in 64 bits.

Weights are whole numbers: a token differs only where a weight was rounded to
another whole number than the reference's and the random number lies within a
few 2^-41 of a border.  The inputs here are fixed, and none does."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module")
def ops(vqx):
    return torch.ops.quantized_ops


def sampled(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, chance, how many are kept) of one row: a list of floats."""
    value = {i: v for i, v in enumerate(x) if v == v and v > -math.inf}
    if not value:
        return -1, -math.inf, 0
    line = sorted(value, key=lambda i: (-value[i], i))
    top = value[line[0]]
    if not t > 0:
        return line[0], 0.0, 1
    w = {i: round(2.0 ** 40 * math.exp(0.0 if value[i] == top else (value[i] - top) / t)) for i in line}
    if 0 < k:
        line = line[:k]
    if p < 1:
        mass, before, kept = sum(w[i] for i in line), 0, []
        for i in line:
            if kept and not float(before) < p * float(mass):
                break
            kept.append(i)
            before += w[i]
        line = kept
    if m > 0:
        line = [i for i in line if float(w[i]) >= min(m, 1.0) * 2.0 ** 40]
    total = sum(w[i] for i in line)
    target = min(max(int(math.floor(u * float(total))), 0), total - 1) if u == u else 0
    for i in sorted(line):
        if target < w[i]:
            return i, math.log(w[i] / total), len(line)
        target -= w[i]


def check(ops, logits, u, t=None, k=None, p=None, m=None):
    f = lambda x, d=torch.float32: None if x is None else torch.tensor(x, dtype=d).to(DEV)  # noqa: E731
    tokens, chances = ops.sample_tokens(logits.to(DEV), f(u), f(t), f(k, torch.int32), f(p), f(m))
    torch.cuda.synchronize()
    assert tokens.dtype == torch.int64 and chances.dtype == torch.float32
    r = lambda x, i, other: other if x is None else float(torch.tensor(x[i], dtype=torch.float32))  # noqa: E731
    kept = []
    for i, row in enumerate(logits.double().tolist()):
        token, chance, n = sampled(row, r(u, i, 0), r(t, i, 1.0), 0 if k is None else k[i], r(p, i, 1.0), r(m, i, 0.0))
        assert int(tokens[i]) == token, f"row {i}: {int(tokens[i])}, not {token}"
        got = float(chances[i])
        # rounded to fp32; a weight of w is off by 1 / w
        assert got == chance or abs(got - chance) <= 2.0 ** -24 * abs(chance) + 2.0 ** -40 * math.exp(-chance) + 2.0 ** -149
        kept.append(n)
    return kept


def rows(n, vocab, kind, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(n, vocab, generator=g)
    return torch.where(torch.rand(n, vocab, generator=g) < 0.02, -math.inf, x).to(TYPES[kind]), torch.rand(n, generator=g).tolist()


VOCABS = [1, 2, 7, 8, 9, 63, 65, 511, 513, 1000, 8191, 8193, 32000, 50257]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("kind", list(TYPES))
def test_all_tokens(ops, vocab, kind):
    x, u = rows(6, vocab, kind, vocab)
    check(ops, x, u)
    check(ops, x, u, t=[0.0, 0.1, 0.7, 1.0, 1.5, 30.0])


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("kind", list(TYPES))
def test_cuts(ops, vocab, kind):
    x, u = rows(8, vocab, kind, vocab + 1)
    t = [0.5, 1.0, 1.0, 0.0, 1.3, 0.8, 1.0, 2.0]
    k = [0, 1, 40, 40, vocab, min(vocab, 300), 7, vocab + 9]
    p = [1.0, 0.9, 0.5, 0.1, 0.99, 0.0, 0.7, 0.95]
    m = [0.0, 0.1, 0.0, 0.3, 0.001, 0.05, 1.0, 0.02]
    check(ops, x, u, t, k)
    check(ops, x, u, t, None, p)
    check(ops, x, u, t, None, None, m)
    check(ops, x, u, None, k, p)
    check(ops, x, u, t, k, p, m)


def test_cuts_keep_more_than_one(ops):
    """What the cuts are for: not all, and not one."""
    x, u = rows(4, 30000, "f32", 3)
    assert check(ops, x, u, None, [50] * 4) == [50] * 4
    assert all(100 < n < 20000 for n in check(ops, x, u, None, None, [0.9] * 4))
    assert all(1 < n < 2000 for n in check(ops, x, u, None, None, None, [0.01] * 4))


@pytest.mark.parametrize("kind", list(TYPES))
def test_equal_logits(ops, kind):
    """Ties go to the lower index, also where thousands are equal, and zeros of
    both signs are."""
    flat = torch.zeros(4, 20000)
    flat[1, ::2] = -0.0
    flat[2] = 3.0
    flat[3, 5000:] = 1.0
    u = [0.999, 0.3, 0.0, 0.5]
    x = flat.to(TYPES[kind])
    check(ops, x, u)
    assert check(ops, x, u, None, [1, 2, 3, 19000]) == [1, 2, 3, 19000]
    check(ops, x, u, None, [12000, 6000, 5000, 16000], [0.5, 0.9, 0.3, 0.99])
    check(ops, x, u, None, None, [0.5, 0.25, 0.75, 0.9])


@pytest.mark.parametrize("kind,k", [("bf16", 9000), ("f32", 9000), ("f16", 5000), ("f32", 31000)])
def test_long_cuts(ops, kind, k):
    """Cuts inside bins with more tokens than are sorted at once: logits that lie
    close together."""
    x, u = rows(3, 40000, kind, 9, spread=0.001)
    check(ops, x, u, None, [k, k + 1, 2 * k])
    check(ops, x, u, None, [k, k + 1, 2 * k], [0.9, 0.5, 0.999])
    check(ops, x, u, [0.5, 1.0, 2.0], None, [0.9, 0.5, 0.999])


@pytest.mark.parametrize("vocab", [4000, 4096, 4097, 8001])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_long_cuts_of_short_rows(ops, vocab, kind):
    """The same where workgroups are smaller: close, equal and ordinary logits."""
    close, u = rows(3, vocab, kind, 9, spread=0.001)
    flat = torch.zeros(3, vocab)
    flat[1, ::2], flat[2, vocab // 4:] = -0.0, 1.0
    k = [vocab // 3, vocab // 2, vocab - 5]
    for x in (close, flat.to(TYPES[kind]), rows(3, vocab, kind, 2)[0]):
        check(ops, x, u, None, k)
        check(ops, x, u, None, k, [0.9, 0.5, 0.999])
        check(ops, x, u, [0.5, 1.0, 2.0], None, [0.9, 0.5, 0.999], [0.0, 0.01, 0.2])


def test_more_rows_than_compute_units(ops):
    """Two workgroups of a compute unit; rows that differ in all they ask for."""
    x, u = rows(520, 8300, "bf16", 5)
    pick = lambda *a: [a[i % len(a)] for i in range(520)]  # noqa: E731
    check(ops, x, u, pick(1.0, 0.7, 0.0, 1.3, 0.9), pick(0, 40, 700, 3000, 1, 8000), pick(1.0, 0.9, 0.99, 0.5), pick(0.0, 0.02, 0.0))


@pytest.mark.parametrize("vocab", [3000, 20000, 600000])
def test_rows_by_themselves(ops, vocab):
    """A row's token does not depend on how many rows are with it, nor then on
    how its work is shared out."""
    g = torch.Generator(DEV).manual_seed(vocab)
    n = 300
    x = (3 * torch.randn(n, vocab, device=DEV, generator=g)).bfloat16()
    f = lambda lo, hi: lo + (hi - lo) * torch.rand(n, device=DEV, generator=g)  # noqa: E731
    u, t, p, m = f(0, 1), f(0.5, 1.5), f(0.5, 1.05), f(-0.01, 0.03)
    k = torch.randint(-2000, 9000, (n,), device=DEV, generator=g).int().clamp(min=0)
    for args in ((t,), (t, k), (t, None, p), (t, k, p, m), (t, None, None, m)):
        want = ops.sample_tokens(x, u, *args)
        for first, end in ((0, 1), (5, 45), (100, 230)):
            got = ops.sample_tokens(x[first:end], u[first:end], *(None if a is None else a[first:end] for a in args))
            assert torch.equal(got[0], want[0][first:end]) and torch.equal(got[1], want[1][first:end]), (len(args), first)


def test_random_numbers_at_the_ends(ops):
    x, _ = rows(7, 999, "f32", 4)
    check(ops, x, [0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan, 1e-30])
    check(ops, x, [0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan, 1e-30], None, [5] * 7, [0.8] * 7)


def test_logits_that_are_not_finite(ops):
    x = torch.randn(9, 300)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 5], x[2, 9] = math.inf, math.inf
    x[3, ::2] = math.nan
    x[4] = -math.inf
    x[4, 77] = -1e30
    x[5] = torch.linspace(-3e38, 3e38, 300)
    x[6, 100] = math.inf
    x[7] = -math.inf
    x[7, 299], x[7, 0] = 1.0, 1.0
    x[8] = torch.where(torch.arange(300) % 3 == 0, 1e-40, -1e-40)
    u = [0.1, 0.2, 0.7, 0.5, 0.9, 0.5, 0.99, 0.6, 0.8]
    for t in (None, [0.0] * 9, [1e-38] * 9, [1e38] * 9):
        for k, p, m in ((None, None, None), ([2] * 9, None, None), (None, [0.6] * 9, [0.5] * 9), ([200] * 9, [0.9] * 9, None)):
            check(ops, x, u, t, k, p, m)


def test_parameters_out_of_range(ops):
    x, u = rows(6, 500, "bf16", 8)
    nan, inf = math.nan, math.inf
    check(ops, x, u, [-1.0, nan, 0.0, 1.0, 1.0, 1.0], [-5, 0, 2 ** 31 - 1, 500, 501, -2 ** 31], [2.0, inf, -1.0, nan, 0.0, -inf],
          [-1.0, 0.0, 2.0, 0.0, -inf, 5.0])


@pytest.mark.parametrize("kind", list(TYPES))
def test_least_weights(ops, kind):
    """Weights of a few units, rounded up to what min_p asks for, and half units."""
    x = torch.full((8, 900), -math.inf).to(TYPES[kind])
    x[:, 5] = 0.0
    for i, z in enumerate((40.9, 40.6, 40.3, 39.7, 39.4, 39.2, 38.9, 41.2)):
        x[i, 700] = -z * math.log(2.0)
    for least in (0.6, 0.9, 1.0, 1.5, 2.0, 2.6, 0.3):
        check(ops, x, [1.0] * 8, m=[least * 2.0 ** -40] * 8)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_logits_further_apart_than_their_type(ops, kind):
    """The largest numbers of both signs, at temperatures that bring them together."""
    x = torch.linspace(-3.3e38, 3.3e38, 700, dtype=torch.float64).repeat(6, 1).to(TYPES[kind])
    u = [0.1, 0.5, 0.9, 0.02, 0.2, 0.999]
    for k, p in ((None, None), ([690] * 6, None), ([1024] * 6, [0.999] * 6), (None, [0.9999] * 6), ([640, 3] * 3, [0.95] * 6)):
        check(ops, x, u, t=[1e38, 2e38, 3e38, 5e37, 3e38, 1e37], k=k, p=p)


def test_small_temperatures(ops):
    """Down to the least number that fp32 has, and logits as near to each other."""
    x = torch.arange(500.0).repeat(6, 1) * torch.tensor([1e-30, 1e-29, 3e-37, 1e-36, 1e-40, 3e-45])[:, None]
    t = [2e-29, 1e-28, 2.0 ** -119, 2.0 ** -120, 2.0 ** -130, 1e-45]
    for k, p in ((None, None), ([40] * 6, None), (None, [0.7] * 6), ([30] * 6, [0.8] * 6)):
        check(ops, x, [0.3] * 6, t=t, k=k, p=p)


def test_distribution(ops):
    """Even numbers give each token its share: of 4096 between its bounds, off by
    at most one on each side."""
    x = torch.tensor([0.0, 1.0, -math.inf, 2.0, 0.5]).repeat(4096, 1)
    u = (torch.arange(4096) + 0.5) / 4096
    tokens, chances = ops.sample_tokens(x.to(DEV), u.to(DEV))
    p = torch.softmax(x[0].double(), -1)
    n = torch.bincount(tokens.cpu(), minlength=5).double()
    assert float((n - 4096 * p).abs().max()) <= 1.0
    assert torch.allclose(chances.cpu().double(), p.log()[tokens.cpu()], rtol=2.0 ** -22)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("start,pad", [(0, 1), (1, 0), (3, 5), (7, 64), (8, 3)])
def test_strided_rows(ops, kind, start, pad):
    """Rows cut out of wider ones start anywhere; what is beside them is not read
    as theirs."""
    x, u = rows(5, 777, kind, 2)
    wide = torch.full((5, start + 777 + pad), 1000.0, dtype=x.dtype)
    wide[:, start:start + 777] = x
    view = wide.to(DEV)[:, start:start + 777]
    k = torch.full((5,), 30, dtype=torch.int32, device=DEV)
    for args in ((), (None, k)):
        got = ops.sample_tokens(view, torch.tensor(u, device=DEV), *args)
        want = ops.sample_tokens(x.to(DEV), torch.tensor(u, device=DEV), *args)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = ops.sample_tokens(x.t().contiguous().to(DEV).t(), torch.tensor(u, device=DEV))
    assert torch.equal(got[0], ops.sample_tokens(x.to(DEV), torch.tensor(u, device=DEV))[0])


def test_broadcast_rows_and_none(ops):
    x, _ = rows(1, 4000, "f32", 6)
    u = torch.rand(40, device=DEV)
    one = ops.sample_tokens(x.to(DEV).expand(40, 4000), u)
    assert torch.equal(one[0], ops.sample_tokens(x.repeat(40, 1).to(DEV), u)[0])
    tokens, chances = ops.sample_tokens(torch.zeros(0, 9, device=DEV), torch.zeros(0, device=DEV))
    assert tokens.shape == chances.shape == (0,)


def test_many_rows_and_a_large_vocabulary(ops):
    x, u = rows(3, 250001, "bf16", 7)
    check(ops, x, u, [1.0, 0.7, 1.2], [1000, 0, 0], [0.95, 0.9, 1.0])
    x, u = rows(700, 50, "f16", 7)
    check(ops, x, u, [0.1 * (i % 20) for i in range(700)], [i % 60 for i in range(700)])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab,start", [(8192, 0), (8193, 3), (32000, 1), (130001, 5), (260000, 0)])
def test_rows_shared_out(ops, kind, vocab, start):
    """Few long rows are shared out over workgroups where no number of tokens
    bounds them; a top_k that keeps all takes the other way to the same tokens."""
    x, u = rows(5, vocab, kind, vocab)
    x[1, 7::3] = -math.inf
    x[2, 100] = x[2, vocab - 1] = math.inf
    x[3, ::2] = math.nan
    x[4] = -math.inf
    wide = torch.full((5, start + vocab + 1), 9.0, dtype=x.dtype)
    wide[:, start:start + vocab] = x
    view, u = wide.to(DEV)[:, start:start + vocab], torch.tensor(u, device=DEV)
    every = torch.zeros(5, dtype=torch.int32, device=DEV)
    f = lambda *v: torch.tensor(v, device=DEV)  # noqa: E731
    for t, p, m in ((None, None, None), (f(1.0, 0.5, 2.0, 1.3, 1.0), None, None), (f(0.0, 0.3, 1.0, 0.0, 1.0), None, None),
                    (None, f(0.9, 0.5, 0.3, 1.0, 0.9), None), (None, None, f(0.01, 0.0, 0.5, 0.3, 0.1)),
                    (f(3.0, 0.2, 1.0, 1.0, 1.0), f(0.99, 0.01, 0.9, 0.0, 0.9), f(0.0, 0.1, 0.0, 1.0, 0.0)),
                    (f(9.0, 9.0, 9.0, 9.0, 9.0), f(0.999, 0.7, 0.9, 0.9, 0.9), None)):
        got, want = ops.sample_tokens(view, u, t, None, p, m), ops.sample_tokens(view, u, t, every, p, m)
        assert torch.equal(got[0], want[0]), (t, p, m)
        assert torch.equal(got[1], want[1])


def test_shared_rows_graph(ops):
    """Captured twice, replayed in turn: the launches of a row share what is theirs."""
    x, u = torch.randn(2, 50000, device=DEV), torch.rand(2, device=DEV)
    p = torch.full((2,), 0.8, device=DEV)
    ops.sample_tokens(x, u, None, None, p)
    graphs = []
    for args in ((None, None, p), ()):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.sample_tokens(x, u, *args)
        graphs.append((graph, out, args))
    for i in range(4):
        x.copy_(torch.randn(2, 50000)), u.copy_(torch.rand(2))
        for graph, out, args in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out, args in graphs:
            want = ops.sample_tokens(x, u, *args)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i


def test_the_same_each_time(ops):
    x, u = rows(16, 60000, "bf16", 11)
    args = (x.to(DEV), torch.tensor(u, device=DEV), None, torch.full((16,), 20000, dtype=torch.int32, device=DEV),
            torch.full((16,), 0.97, device=DEV))
    first = ops.sample_tokens(*args)
    for _ in range(5):
        again = ops.sample_tokens(*args)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_sampling_graph(ops):
    """A captured draw follows logits, numbers and parameters as they change."""
    x, u, t = torch.randn(8, 5000, device=DEV), torch.rand(8, device=DEV), torch.ones(8, device=DEV)
    k, p = torch.full((8,), 50, dtype=torch.int32, device=DEV), torch.full((8,), 0.9, device=DEV)
    ops.sample_tokens(x, u, t, k, p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_tokens(x, u, t, k, p)
    for i in range(4):
        x.copy_(torch.randn(8, 5000)), u.copy_(torch.rand(8)), t.fill_(0.5 + 0.3 * i), k.fill_(10 + i), p.fill_(0.8 + 0.05 * i)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.sample_tokens(x, u, t, k, p)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
