"""Attention of drafted tokens over the 4-bit cache, against a 64-bit form."""

import math
import random

import pytest
import torch

from tests import kv4_reference as ref
from tests.test_gpu_kv4 import TYPES, WEIGHT, make_cache, near, on, same
from tests.test_gpu_kv4_pages import forest, signed

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module")
def ops(vqx):
    return torch.ops.quantized_ops


def distances(mask, count, base, tokens):
    """Of each token that the row sees, how far before it it is: a list of -1s
    and distances."""
    line = [j for j in range(count) if mask >> j & 1]
    away = [base + len(line) - 1 - t if t < base else -1 for t in range(tokens)]
    for back, j in enumerate(reversed(line)):
        if 0 <= base + j < tokens:
            away[base + j] = back
    return away


def attention(q, codes, scales, lengths, tree, cu=None, table=None, scale=None, softcap=0.0, window=0, slopes=None):
    """(out, lse, size of what an output sums, how far a score may be off in fp32
    with queries held to 2^-22 of their largest), as kv4_reference has it."""
    n, heads, dim = q.shape
    pages, kv, size = codes.shape[1:4]
    group = heads // kv
    scale = dim ** -0.5 if scale is None else scale
    q = q.double()
    out, mass = torch.zeros(n, heads, dim).double(), torch.zeros(n, heads, dim).double()
    lse, err = torch.full((n, heads), -math.inf).double(), torch.zeros(n, heads).double()
    for b, (first, end) in enumerate(ref.spans(n, lengths.shape[0], cu)):
        tokens = max(0, min(int(lengths[b]), ref.room(codes, table)))
        where = ref.places(table, size, pages, b, range(tokens))
        if not where or first == end:
            continue
        t, page, slot = (torch.tensor(x) for x in zip(*where))
        away = torch.tensor([distances(tree[i], end - first, int(lengths[b]) - (end - first), tokens)
                             for i in range(first, end)])[:, t]
        seen = (away >= 0) & ((away < window) if window else True)
        for h in range(kv):
            k, v = (ref.decode(codes[i][page, h, slot], scales[i][page, h, slot]) for i in (0, 1))
            for x in range(h * group, (h + 1) * group):
                rows = q[first:end, x]
                a = rows @ k.T * scale
                if softcap:
                    a = softcap * torch.tanh(a / softcap)
                if slopes is not None:
                    a = a - slopes[x].double() * away
                a = a.masked_fill(~seen, -math.inf)
                z = torch.logsumexp(a, -1)
                p = torch.where(seen, torch.exp(a - z[:, None]), 0.0)
                lse[first:end, x] = z
                # a NaN value matters to the rows that see it, also at weight 0
                nan = (seen.double() @ v.isnan().double()) > 0
                out[first:end, x] = (p @ v.nan_to_num()).masked_fill(nan, math.nan)
                mass[first:end, x] = p @ v.abs().nan_to_num()
                s = a.masked_fill(~seen, 0.0).nan_to_num()
                e = abs(scale) * ((dim + 4) * 2.0 ** -24 * (rows.abs() @ k.abs().nan_to_num().T).amax(-1)
                                  + 2.0 ** -22 * rows.abs().amax(-1) * k.abs().nan_to_num().sum(-1).max())
                e = e + 8 * 2.0 ** -24 * (s.abs().amax(-1) + softcap)
                if slopes is not None:
                    e = e + 4 * 2.0 ** -24 * slopes[x].abs() * away.amax(-1)
                err[first:end, x] = e
    return out, lse, mass, err


def check(ops, kind, q, codes, scales, lengths, tree, cu=None, most=None, table=None, live=None, **how):
    masks = torch.tensor([signed(m) for m in tree], dtype=torch.int64)
    dq, dc, ds, dl, dm, dcu, dt = on(q, codes, scales, lengths, masks, cu, table)
    slopes = how.get("slopes")
    out, lse = ops.kv4_tree_attention(dq, dc, ds, dl, dm, dcu, most, dt,
                                      **dict(how, slopes=None if slopes is None else slopes.to(DEV)))
    torch.cuda.synchronize()
    w_out, w_lse, mass, err = attention(q, codes, scales, lengths, tree, cu, table, **how)
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    n = live if live is not None else q.shape[0]
    out, lse, w_out, w_lse, mass, err = (t[:n] for t in (out, lse, w_out, w_lse, mass, err))
    # twice a score's error on a weight and its sum, sums of fp32 in some order,
    # the weights' terms, the output's half step
    rel = 2 * err + 64 * 2.0 ** -24
    tol = torch.finfo(q.dtype).eps / 2 * w_out.abs() + (rel[..., None] + WEIGHT[kind]) * (1 + 2.0 ** -8) * mass + 1e-30
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    near(out, w_out, tol, "out")
    near(lse, w_lse, err + 64 * 2.0 ** -24 + 8 * 2.0 ** -24 * w_lse.abs().nan_to_num(0, 0, 0), "lse")
    return out, lse


def scene(kind, dim, kv, group, lengths, news, page, seed=0):
    g = torch.Generator().manual_seed(seed + dim)
    codes, scales, table = make_cache(len(lengths), kv, dim, max(lengths + [1]), page, seed)
    q = torch.randn(sum(news), kv * group, dim, generator=g).to(TYPES[kind])
    return q, codes, scales, torch.tensor(lengths).int(), torch.tensor([0] + news).cumsum(0).int(), table


CASES = [
    # kind, dim, kv, group, lengths, new tokens, page, how
    ("bf16", 128, 2, 4, [1, 40, 300], [1, 7, 12], 0, {}),
    ("bf16", 128, 2, 4, [64, 65, 700, 9], [64, 64, 33, 0], 16, {}),
    ("f16", 64, 1, 5, [130, 31, 2000], [9, 31, 64], 48, dict(softcap=20.0)),
    ("f32", 64, 3, 1, [77, 8], [7, 8], 0, {}),
    ("f32", 256, 1, 2, [90, 33], [20, 33], 32, dict(window=5)),
    ("bf16", 256, 2, 1, [200, 64, 5], [30, 1, 5], 7, dict(window=40)),
    ("bf16", 64, 1, 8, [500, 64], [50, 64], 64, dict(window=20, slopes=True)),
    ("f16", 128, 4, 2, [333, 100, 64], [17, 40, 64], 100, dict(slopes=True, softcap=30.0)),
    ("f32", 128, 1, 3, [150, 5000], [25, 3], 16, dict(slopes=True, scale=-0.2)),
    ("bf16", 128, 8, 1, [20000, 600], [4, 60], 256, {}),
]


@pytest.mark.parametrize("kind,dim,kv,group,lengths,news,page,how", CASES)
@pytest.mark.parametrize("seed", [0, 1])
def test_tree(ops, kind, dim, kv, group, lengths, news, page, how, seed):
    s = scene(kind, dim, kv, group, lengths, news, page, seed)
    if how.get("slopes"):
        how = dict(how, slopes=torch.linspace(0.01, 0.5, kv * group))
    check(ops, kind, *s[:4], forest(news, seed)[0], s[4], max(news), s[5], **how)


# 16 kv heads of 8 query heads: workgroups of many rows, in every type and size
@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("f16", 64), ("f32", 128), ("bf16", 256), ("f32", 64), ("f16", 256)])
@pytest.mark.parametrize("how", [{}, dict(softcap=15.0, window=33, slopes=True)])
@pytest.mark.parametrize("page", [0, 24])
def test_tree_many_rows(ops, kind, dim, how, page):
    lengths, news = [100, 64, 200, 90, 65, 150, 71, 80], [64, 64, 60, 33, 64, 64, 1, 50]
    s = scene(kind, dim, 16, 8, lengths, news, page)
    if how.get("slopes"):
        how = dict(how, slopes=torch.linspace(0.01, 0.5, 128))
    check(ops, kind, *s[:4], forest(news, 2)[0], s[4], 64, s[5], **how)


@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("f16", 64), ("f32", 128), ("bf16", 256), ("f32", 64), ("f16", 256)])
@pytest.mark.parametrize("how", [{}, dict(softcap=15.0, window=33, slopes=True)])
@pytest.mark.parametrize("page", [0, 24])
def test_tree_full_tiles(ops, kind, dim, how, page):
    """Almost all of the workgroups' rows are there: those of many rows."""
    lengths, news = [100, 64, 200, 90, 65, 150, 71, 480], [64, 64, 60, 64, 57, 64, 64, 64]
    s = scene(kind, dim, 16, 8, lengths, news, page)
    if how.get("slopes"):
        how = dict(how, slopes=torch.linspace(0.01, 0.5, 128))
    check(ops, kind, *s[:4], forest(news, 2)[0], s[4], 64, s[5], **how)


@pytest.mark.parametrize("how", [{}, dict(slopes=True)])
def test_tree_full_tiles_in_parts(ops, how):
    """The same over a long sequence, in parts that are joined."""
    s = scene("bf16", 64, 4, 8, [25100], [64], 128)
    if how.get("slopes"):
        how = dict(slopes=torch.linspace(0.0001, 0.005, 32))
    check(ops, "bf16", *s[:4], forest([64], 5)[0], s[4], 64, s[5], **how)


@pytest.mark.parametrize("seqs", [63, 64, 65])
def test_tree_of_sequences_by_length(ops, seqs):
    """Workgroups in the order of lengths, some of them equal or 0, up to 64
    sequences."""
    news = [1 + (5 * b) % 7 for b in range(seqs)]
    lengths = [max((37 * b) % 90 // 4 * 4, news[b]) for b in range(seqs)]
    s = scene("bf16", 64, 4, 4, lengths, news, 16)
    given = s[3].clone()
    given[::9] = 0  # nothing of these is there
    check(ops, "bf16", *s[:3], given, forest(news, 1)[0], s[4], max(news), s[5])


@pytest.mark.parametrize("kv,group,news", [(2, 4, [12, 1, 40]), (16, 8, [64, 64, 60])])
@pytest.mark.parametrize("how", [dict(softcap=20.0), dict(slopes=True)])
def test_a_chain_is_a_prompt(ops, kv, group, news, how):
    """Tokens one after another: kv4_attention's own rows, bit for bit where that
    caps or slopes its scores too."""
    q, codes, scales, lengths, cu, table = on(*scene("bf16", 128, kv, group, [90, 300, 64], news, 16))
    if how.get("slopes"):
        how = dict(slopes=torch.linspace(0.01, 0.5, kv * group, device=DEV))
    masks = torch.tensor([signed((2 << j) - 1) for c in news for j in range(c)], device=DEV)
    got = ops.kv4_tree_attention(q, codes, scales, lengths, masks, cu, max(news), table, **how)
    want = ops.kv4_attention(q, codes, scales, lengths, cu, max(news), table, **how)
    same(got[0], want[0].cpu(), "out")
    same(got[1], want[1].cpu(), "lse")


def test_any_masks(ops):
    """Masks that are no tree: nothing set, all set (bits of tokens that are not
    there too), tokens behind a row's own."""
    r = random.Random(5)
    news = [9, 64, 20]
    tree = [r.choice([0, 2 ** 64 - 1, r.getrandbits(64), 1 << r.randrange(64)]) for _ in range(sum(news))]
    for how in ({}, dict(window=6), dict(slopes=torch.linspace(0.1, 1.0, 8))):
        s = scene("f32", 64, 2, 4, [50, 64, 300], news, 16)
        check(ops, "f32", *s[:4], tree, s[4], 64, s[5], **how)


def test_rows_that_see_nothing(ops):
    """No cached tokens and no bits: 0 and -inf."""
    s = scene("bf16", 128, 1, 4, [6, 3], [6, 3], 0)
    tree = [1, 0, 3, 0, 0, 9, 0, 0, 0]
    out, lse = check(ops, "bf16", *s[:4], tree, s[4], 6, s[5])
    assert bool((out[[1, 3, 4, 6, 7, 8]] == 0).all()) and bool((lse[[1, 3, 4, 6, 7, 8]] == -math.inf).all())


def test_places_before_the_beginning(ops):
    """A length below the number of new tokens: the first of them are nowhere."""
    news = [12, 20]
    s = scene("f32", 64, 2, 2, [5, 40], news, 16)
    check(ops, "f32", *s[:3], torch.tensor([5, 0]).int(), forest(news, 1)[0], s[4], 20, s[5])


def test_missing_pages_and_full_rooms(ops):
    news = [30, 40]
    q, codes, scales, lengths, cu, table = scene("f16", 128, 2, 2, [100, 200], news, 16)
    table[0, 5], table[1, 3], table[1, 11] = -1, 10 ** 6, -7
    check(ops, "f16", q, codes, scales, torch.tensor([100, 230]).int(), forest(news, 3)[0], cu, 40, table)


def test_nan_and_large_values_that_are_not_seen(ops):
    """A drafted token's NaN keys and values reach its descendants only."""
    news = [24, 8]
    for kind in ("bf16", "f32"):
        q, codes, scales, lengths, cu, table = scene(kind, 128, 2, 4, [60, 40], news, 16)
        tree = forest(news, 7)[0]
        for b, j, plane, byte in ((0, 5, 0, 255), (0, 9, 1, 255), (1, 2, 1, 254), (1, 3, 0, 255)):
            t = int(lengths[b]) - news[b] + j
            scales[plane, table[b, t // 16], :, t % 16, 1] = byte
        masks = torch.tensor([signed(m) for m in tree])
        dev = on(q, codes, scales, lengths, masks, cu)
        out, lse = ops.kv4_tree_attention(*dev, 24, table.to(DEV))
        w_out, w_lse, _, _ = attention(q, codes, scales, lengths, tree, cu, table)
        hit = torch.tensor([bool(tree[i] >> 5 & 1) if i < 24 else bool(tree[i] >> 3 & 1) for i in range(32)])
        assert 0 < int(hit.sum()) < 32
        assert torch.equal(lse.isnan().any(-1).cpu(), hit), "NaN keys"
        spared = ~hit & ~w_out.isnan().any(-1).any(-1)
        assert bool(out.cpu()[spared].isfinite().all())
        clean = torch.tensor([not (tree[i] >> 2 & 1) if i >= 24 else True for i in range(32)]) & spared
        near(out.cpu()[clean], w_out[clean], 2.0 ** -7 * w_out[clean].abs() + 2.0 ** -7, "out")
        want_nan = torch.tensor([bool(tree[i] >> 9 & 1) and i < 24 for i in range(32)]) & ~hit
        assert bool(out.cpu()[want_nan][..., 32:64].isnan().all()) and bool(out.cpu()[want_nan][..., 64:].isfinite().all())


def test_more_new_tokens_than_most(ops):
    """Rows beyond the most that the call was told of have NaN."""
    news = [70, 20]
    s = scene("f32", 64, 1, 2, [90, 40], news, 16)
    tree = forest(news, 1)[0]
    dev = on(*s[:4], torch.tensor([signed(m) for m in tree]), s[4])
    out, lse = ops.kv4_tree_attention(*dev, 64, s[5].to(DEV))
    assert bool(out[64:70].isnan().all()) and bool(lse[64:70].isnan().all())
    assert bool(out[:64].isfinite().all()) and bool(out[70:].isfinite().all())
    w_out = attention(*s[:4], tree, s[4], s[5])[0]
    near(out[70:], w_out[70:], 2.0 ** -18 * (1 + w_out[70:].abs()), "the other sequence")


def test_even_offsets_and_strides(ops):
    """As many for each sequence; queries cut out of a projection."""
    q, codes, scales, lengths, _, table = scene("bf16", 128, 2, 4, [50, 9, 200], [9, 9, 9], 16)
    wide = torch.randn(27, 12, 128).bfloat16()
    wide[:, 2:10] = q
    tree = forest([9, 9, 9], 4)[0]
    check(ops, "bf16", wide[:, 2:10], codes, scales, lengths, tree, None, None, table)


def test_no_new_tokens(ops):
    q, codes, scales, lengths, cu, table = on(*scene("bf16", 128, 2, 4, [50, 9], [0, 0], 16))
    out, lse = ops.kv4_tree_attention(q, codes, scales, lengths, torch.zeros(0, dtype=torch.int64, device=DEV), cu, None, table)
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)


def test_tree_graph(ops):
    """A captured step follows masks, queries and lengths as they change."""
    news = [20, 33, 1]
    q, codes, scales, lengths, cu, table = on(*scene("bf16", 128, 2, 4, [2000, 400, 64], news, 64))
    masks = torch.zeros(54, dtype=torch.int64, device=DEV)
    call = lambda: ops.kv4_tree_attention(q, codes, scales, lengths, masks, cu, 33, table)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in range(4):
        masks.copy_(torch.tensor([signed(m) for m in forest(news, seed)[0]]))
        q.copy_(torch.randn(q.shape))
        lengths.copy_(torch.tensor([1990 - seed, 400 - 40 * seed, 64]))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, call()):
            same(got, want.cpu(), f"replay {seed}")
