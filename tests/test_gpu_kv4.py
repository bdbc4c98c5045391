"""The 4-bit cache's operators on the GPU against plain 64-bit forms."""

import math

import pytest
import torch

from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# a weight's rounding in the product with the values, at most
WEIGHT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -16, "f32": 2.0 ** -24}


@pytest.fixture(scope="module")
def ops(vqx):
    return torch.ops.quantized_ops


def make_cache(seqs, kv, dim, room, page, seed=0, spare=2):
    """(codes, scales, table) on the CPU, all bytes random."""
    g = torch.Generator().manual_seed(seed)
    if page:
        each = -(-room // page)
        pages, size = seqs * each + spare, page
        table = torch.randperm(pages, generator=g)[:seqs * each].reshape(seqs, each).int()
    else:
        pages, size, table = seqs, room, None
    codes = torch.randint(0, 256, (2, pages, kv, size, dim // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(123, 128, (2, pages, kv, size, dim // 32), generator=g, dtype=torch.uint8)
    return codes, scales, table


def on(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def same(got, want, what):
    off = int((got.cpu() != want.cpu()).sum())
    assert off == 0, f"{what}: {off} of {want.numel()} differ"


def near(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities"
    ok = ~(want.isnan() | inf)
    off = ((got - want).abs() - tol)[ok]
    assert off.numel() == 0 or float(off.max()) <= 0, \
        f"{what}: off by {float((got - want).abs()[ok].max())}, {int((off > 0).sum())} of {off.numel()} too far"


def check_attention(ops, kind, q, codes, scales, lengths, cu=None, most=None, table=None, weigh=True, **how):
    dq, dc, ds, dl, dcu, dt = on(q, codes, scales, lengths, cu, table)
    slopes = how.get("slopes")
    dhow = dict(how, slopes=None if slopes is None else slopes.to(DEV))
    out, lse = ops.kv4_attention(dq, dc, ds, dl, dcu, most, dt, **dhow)
    torch.cuda.synchronize()
    w_out, w_lse, added, mass, err = ref.attention(q, codes, scales, lengths, cu, table, **how)
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    # twice a score's error on a weight and its sum, sums of fp32 in some order,
    # the weights' terms, the output's half step
    rel = 2 * err + 64 * 2.0 ** -24
    tol = torch.finfo(q.dtype).eps / 2 * w_out.abs() + (rel[..., None] + WEIGHT[kind]) * (1 + 2.0 ** -8) * mass + 1e-30
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    near(out, w_out, tol, "out")
    near(lse, w_lse, err + 64 * 2.0 ** -24 + 8 * 2.0 ** -24 * w_lse.abs().nan_to_num(0, 0, 0), "lse")
    if weigh:
        w = torch.rand(added.shape, generator=torch.Generator().manual_seed(5))
        dw = w.to(DEV)
        ops.kv4_accumulate(dq, lse, dc, ds, dl, dw, dcu, most, dt, **dhow)
        # lse has its own error, once more
        e = float(err.max()) * 3 + 128 * 2.0 ** -24 + 16 * 2.0 ** -24 * float(w_lse.abs().nan_to_num(0, 0, 0).max())
        near(dw, w.double() + added, e * added + 2.0 ** -23 * (w.double() + added), "weights")
    return out, lse


CASES = [
    # kind, dim, kv, group, lengths, new, page, how
    ("bf16", 128, 2, 4, [1, 2, 31, 32, 33], 1, 0, {}),
    ("bf16", 128, 2, 4, [0, 1, 127, 128, 129, 700], 1, 16, {}),
    ("bf16", 64, 3, 1, [77, 5, 64], 1, 0, {}),
    ("f16", 64, 1, 5, [1000, 3], 1, 48, {}),
    ("f32", 64, 4, 3, [77], 1, 0, {}),
    ("f32", 128, 1, 8, [2051, 1300], 1, 64, {}),
    ("f16", 128, 2, 2, [513, 1025], 1, 7, {}),
    ("bf16", 256, 2, 2, [40, 333], 1, 32, {}),
    ("f16", 256, 1, 1, [95], 1, 0, {}),
    ("f32", 256, 1, 20, [130, 7], 1, 5, {}),
    ("bf16", 128, 1, 4, [300, 40], 37, 64, {}),
    ("f16", 64, 2, 8, [200, 33], 9, 16, {}),
    ("f32", 256, 1, 2, [70, 50], 50, 0, {}),
    ("bf16", 128, 2, 1, [300], 300, 0, {}),
    ("bf16", 64, 1, 16, [90, 64], 65, 1, {}),
    ("bf16", 128, 1, 3, [400, 130], 5, 64, dict(window=100)),
    ("f16", 128, 1, 3, [400, 30], 70, 64, dict(window=33)),
    ("f32", 64, 2, 2, [300, 30], 17, 0, dict(window=1)),
    ("bf16", 64, 2, 4, [300, 30], 17, 16, dict(softcap=30.0)),
    ("f32", 128, 2, 2, [300, 30], 1, 0, dict(softcap=2.0)),
    ("f16", 256, 1, 4, [150, 30], 3, 32, dict(softcap=50.0, window=64)),
    ("bf16", 128, 2, 4, [2100, 30], 1, 64, dict(slopes=True)),
    ("f32", 64, 1, 4, [1500, 30], 4, 24, dict(slopes=True, softcap=20.0, window=700)),
    ("bf16", 128, 1, 2, [200], 3, 0, dict(scale=-0.3)),
    ("bf16", 128, 1, 2, [200], 3, 0, dict(scale=0.0)),
]


@pytest.mark.parametrize("i", range(len(CASES)), ids=lambda i: "-".join(map(str, CASES[i][:4])) + f"-new{CASES[i][5]}"
                         f"-page{CASES[i][6]}" + "".join(f"-{k}" for k in CASES[i][7]))
def test_attention(ops, i):
    kind, dim, kv, group, lens, new, page, how = CASES[i]
    print("case", CASES[i], flush=True)
    g = torch.Generator().manual_seed(i)
    heads, seqs = kv * group, len(lens)
    codes, scales, table = make_cache(seqs, kv, dim, max(lens), page, i)
    q = torch.randn(seqs * new, heads, dim, generator=g).to(TYPES[kind])
    how = dict(how)
    if how.get("slopes"):
        how["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads + 1) / heads)
    check_attention(ops, kind, q, codes, scales, torch.tensor(lens, dtype=torch.int32), table=table, **how)


def widened(codes, scales, table, tiles):
    """The same cache with room for so many tokens that a call of `tiles` tiles
    of 16 rows, over all sequences and kv heads, is one for many rows (200000
    tiles of 16 rows by 32 tokens at most): a table of pages that are none, or longer
    sequences."""
    room = -(-200000 // tiles) * 32 + 64
    if table is not None:
        more = room // codes.shape[3] + 1 - table.shape[1]
        return codes, scales, torch.nn.functional.pad(table, (0, max(0, more)), value=-1)
    pad = (0, 0, 0, max(0, room - codes.shape[3]))
    return torch.nn.functional.pad(codes, pad), torch.nn.functional.pad(scales, pad), None


MANY = [i for i, c in enumerate(CASES) if c[3] * c[5] > 16] + [
    ("bf16", 128, 2, 4, [500, 130, 64], 61, 64, {}), ("bf16", 128, 1, 2, [1000, 400], 150, 128, {}),
    ("bf16", 64, 1, 5, [300, 63], 40, 256, dict(softcap=3.0)), ("f16", 128, 1, 4, [129, 190], 33, 64, dict(slopes=True)),
    ("f32", 128, 2, 1, [200, 90], 80, 64, dict(window=50, softcap=9.0)), ("f32", 64, 1, 3, [333], 100, 0, {}),
    ("bf16", 256, 1, 3, [140, 70], 50, 64, dict(window=64)), ("f16", 256, 1, 2, [200], 90, 16, dict(softcap=30.0)),
    ("f32", 256, 1, 2, [150], 70, 64, dict(slopes=True)), ("bf16", 128, 1, 4, [70], 70, 0, dict(scale=-0.2)),
    ("bf16", 128, 1, 40, [3, 33], 1, 64, {})]


@pytest.mark.parametrize("i", range(len(MANY)))
def test_attention_many_rows(ops, i):
    """The kernel for many rows, at small sizes: what takes it is the room."""
    kind, dim, kv, group, lens, new, page, how = CASES[MANY[i]] if isinstance(MANY[i], int) else MANY[i]
    print("case", (kind, dim, kv, group, lens, new, page, how), flush=True)
    g = torch.Generator().manual_seed(i)
    heads, seqs = kv * group, len(lens)
    codes, scales, table = make_cache(seqs, kv, dim, max(lens), page, i)
    codes, scales, table = widened(codes, scales, table, seqs * kv * -(-new * group // 16))
    q = torch.randn(seqs * new, heads, dim, generator=g).to(TYPES[kind])
    how = dict(how)
    if how.get("slopes"):
        how["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads + 1) / heads)
    if how.get("window"):
        # a window bounds what a tile can see: more sequences, that have nothing
        more = -(-200000 * 32 // (kv * -(-new * group // 16) * (how["window"] + new)))
        lens = lens + [0] * more
        q = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, new * more))
        if table is not None:
            table = torch.nn.functional.pad(table[:, :64], (0, 0, 0, more), value=-1)
        else:
            codes, scales = (torch.nn.functional.pad(x[..., :max(lens), :], (0, 0, 0, 0, 0, 0, 0, more)) for x in (codes, scales))
    check_attention(ops, kind, q, codes, scales, torch.tensor(lens, dtype=torch.int32), table=table, weigh=False, **how)


@pytest.mark.parametrize("page", [0, 48, 64])
def test_attention_many_rows_and_heads(ops, page):
    """As many tiles as need no splits: outputs straight from the kernel."""
    g = torch.Generator().manual_seed(page)
    seqs, kv, group, dim, new = 65, 8, 2, 64, 20
    lens = torch.randint(1, 90, (seqs,), generator=g).int()
    lens[0] = 90
    codes, scales, table = widened(*make_cache(seqs, kv, dim, 90, page), seqs * kv * 3)
    q = torch.randn(seqs * new, kv * group, dim, generator=g).bfloat16()
    check_attention(ops, "bf16", q, codes, scales, lens, table=table, weigh=False)


@pytest.mark.parametrize("page", [8, 64])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_many_rows_nan_and_bad_pages(ops, dim, page):
    new = 20
    codes, scales, table = make_cache(3, 1, dim, 128, page)
    for t, plane, block in ((80, 1, 0), (88, 1, dim // 32 - 1), (95, 0, 0), (3, 1, 1)):
        _, p, slot = ref.places(table, codes.shape[3], codes.shape[1], 0, [t])[0]
        scales[plane, p, 0, slot, block] = 255
    table[1, 0], table[2, 1] = -1, codes.shape[1]
    codes, scales, table = widened(codes, scales, table, 3 * 3)
    q = torch.randn(3 * new, 2, dim, generator=torch.Generator().manual_seed(1)).bfloat16()
    lens = torch.tensor([96, 100, 128], dtype=torch.int32)
    out, lse = check_attention(ops, "bf16", q, codes, scales, lens, table=table, weigh=False)
    assert not lse[:19].isnan().any() and lse[19].isnan().all()
    assert not out[:4].isnan()[..., 64:].any() and not out[new:].isnan().any()


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 0)])
def test_attention_many_rows_of_values_of_many_sizes(ops, dim, page):
    """Scales that grow along a sequence, zeros with the smallest scale, and a
    page that is none over one that holds the largest of all."""
    codes, scales, table = make_cache(2, 1, dim, 400, page)
    for t, byte in ((5, 110), (6, 131), (70, 113), (71, 100), (130, 0), (201, 134), (399, 145)):
        _, p, slot = ref.places(table, codes.shape[3], codes.shape[1], 0, [t])[0]
        scales[1, p, 0, slot, 1] = byte
        if byte == 0:
            codes[1, p, 0, slot] = 0
    if page:
        codes, scales, table = (torch.cat([x[:, :1], x], 1) if i < 2 else x + 1 for i, x in enumerate((codes, scales, table)))
        scales[1, 0] = 254  # what a token without a page reads
        table[1, 1] = -1
    codes, scales, table = widened(codes, scales, table, 2 * 8)
    q = torch.randn(2 * 40, 3, dim, generator=torch.Generator().manual_seed(1)).bfloat16()
    check_attention(ops, "bf16", q, codes, scales, torch.tensor([400, 100], dtype=torch.int32), table=table, weigh=False)


def test_attention_many_rows_ragged(ops):
    new, most = [0, 1, 70, 9, 0, 130], 100
    lens = torch.tensor([40, 300, 170, 4, 0, 140], dtype=torch.int32)
    cu = torch.tensor([0] + new).cumsum(0).int()
    codes, scales, table = widened(*make_cache(6, 2, 128, 300, 16), 6 * 2 * 19)
    q = torch.randn(sum(new), 6, 128, generator=torch.Generator().manual_seed(3)).bfloat16()
    out, lse = check_attention(ops, "bf16", q, codes, scales, lens, cu, None, table, weigh=False)
    d = on(q, codes, scales, lens, cu, table)
    short, short_lse = ops.kv4_attention(d[0], d[1], d[2], d[3], d[4], most, d[5])
    assert short[80 + most:].isnan().all() and short_lse[80 + most:].isnan().all()
    near(short[:80 + most], out[:80 + most].cpu().double(), 2.0 ** -7 * out[:80 + most].cpu().double().abs() + 2.0 ** -6, "most")


@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("f16", 64), ("f32", 256)])
@pytest.mark.parametrize("most", [None, 70, 200])
def test_attention_ragged(ops, kind, dim, most):
    """Sequences with 0, 1 and many new tokens; one has more of them than tokens."""
    g = torch.Generator().manual_seed(3)
    new = [0, 1, 70, 9, 0]
    lens = torch.tensor([40, 300, 170, 4, 0], dtype=torch.int32)
    cu = torch.tensor([0] + new).cumsum(0).int()
    codes, scales, table = make_cache(5, 2, dim, 300, 16)
    q = torch.randn(sum(new), 6, dim, generator=g).to(TYPES[kind])
    out, lse = check_attention(ops, kind, q, codes, scales, lens, cu, most, table)
    assert torch.equal(lse[71:76].cpu(), torch.full((5, 6), -math.inf)) and not out[71:76].any()


@pytest.mark.parametrize("kind,dim,page", [("bf16", 128, 16), ("f16", 64, 0), ("f32", 256, 48)])
@pytest.mark.parametrize("new,lens,kv,many", [
    ([1] * 37 + [100] + [1] * 35 + [5], [20 + i for i in range(37)] + [130] + [3 * i for i in range(36)], 3, False),
    ([0, 1, 120, 1, 0, 2, 1], [0, 1700, 2000, 5, 900, 2, 1000], 1, False),
    ([3, 0, 300, 0], [40, 7, 310, 0], 2, True),
    ([0, 130, 2], [800, 5000, 70], 1, True),
])
def test_attention_mixed(ops, kind, dim, page, new, lens, kv, many):
    """Few sequences with many new tokens among others with one or none: the
    tiles that there are come one after another, over more than a wave's
    sequences, with splits and without."""
    cu = torch.tensor([0] + new).cumsum(0).int()
    lens = torch.tensor(lens, dtype=torch.int32)
    codes, scales, table = make_cache(len(new), kv, dim, int(lens.max()), page)
    if many:
        codes, scales, table = widened(codes, scales, table, sum(new) * 4 * kv // 16)
    q = torch.randn(sum(new), kv * 4, dim, generator=torch.Generator().manual_seed(len(new))).to(TYPES[kind])
    check_attention(ops, kind, q, codes, scales, lens, cu, max(new), table)


def test_attention_mixed_more_than_most(ops):
    """Offsets with more new tokens than `most`, out of order and past the end:
    rows of sound sequences are right, the others' are NaN or left alone."""
    new = [1, 1, 40, 1, 1, 1, 1, 1]
    cu = torch.tensor([0] + new).cumsum(0).int()
    lens = torch.full((8,), 60, dtype=torch.int32)
    codes, scales, table = make_cache(8, 2, 128, 64, 16)
    q = torch.randn(sum(new), 8, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    d = on(q, codes, scales, lens, cu, table)
    want, want_lse = ops.kv4_attention(d[0], d[1], d[2], d[3], d[4], 40, d[5])
    out, lse = ops.kv4_attention(d[0], d[1], d[2], d[3], d[4], 30, d[5])
    assert out[32:42].isnan().all() and lse[32:42].isnan().all()
    got, want = torch.cat([out[:32], out[42:]]), torch.cat([want[:32], want[42:]]).cpu().double()
    near(got, want, 2.0 ** -7 * want.abs() + 2.0 ** -6, "out")
    cu[4:] = torch.tensor([1 << 30, -5, 1 << 30, 47, 0], dtype=torch.int32)
    ops.kv4_attention(d[0], d[1], d[2], d[3], cu.to(DEV), 40, d[5])
    torch.cuda.synchronize()


def test_attention_of_more_than_most(ops):
    """Queries past `most` come back as NaN, the others as they are."""
    codes, scales, table = on(*make_cache(2, 1, 128, 64, 32))
    q = torch.randn(12, 2, 128, device=DEV).bfloat16()
    lens, cu = torch.tensor([64, 40], dtype=torch.int32, device=DEV), torch.tensor([0, 9, 12], dtype=torch.int32, device=DEV)
    out, lse = ops.kv4_attention(q, codes, scales, lens, cu, 5, table)
    all_out, _ = ops.kv4_attention(q, codes, scales, lens, cu, None, table)
    assert out[5:9].isnan().all() and lse[5:9].isnan().all()
    assert torch.equal(out[:5], all_out[:5]) and torch.equal(out[9:], all_out[9:])


@pytest.mark.parametrize("page", [16, 32])
def test_attention_bad_pages(ops, page):
    """Tokens on an entry that is no page are not attended to, wherever it lies."""
    codes, scales, table = make_cache(3, 2, 128, 160, page)
    table[0, 1], table[1, 0], table[2, :] = -1, codes.shape[1], 2 ** 31 - 1
    q = torch.randn(6, 4, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    out, lse = check_attention(ops, "bf16", q, codes, scales, torch.tensor([160, 33, 20], dtype=torch.int32), table=table)
    assert not out[4:].any() and bool((lse[4:] == -math.inf).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [0, 8])
def test_attention_nan_values(ops, dim, page):
    """A NaN block of values reaches the rows that see it, in its own elements;
    a NaN key all of a row; and neither reaches a row that does not see it."""
    new = 20
    codes, scales, table = make_cache(2, 1, dim, 96, page)
    for t, plane, block in ((80, 1, 0), (88, 1, dim // 32 - 1), (92, 0, 0), (3, 1, 1)):
        _, p, slot = ref.places(table, codes.shape[3], codes.shape[1], 0, [t])[0]
        scales[plane, p, 0, slot, block] = 255
    q = torch.randn(2 * new, 2, dim, generator=torch.Generator().manual_seed(1)).bfloat16()
    lens = torch.tensor([96, 50], dtype=torch.int32)
    out, lse = check_attention(ops, "bf16", q, codes, scales, lens, table=table, window=30, weigh=False)
    assert not lse[:16].isnan().any() and lse[16:20].isnan().all()
    assert not out[new:].isnan().any()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_attention_of_a_query_that_is_not_finite(ops, bad):
    codes, scales, _ = on(*make_cache(1, 1, 128, 40, 0))
    q = torch.randn(1, 4, 128, device=DEV).bfloat16()
    lens = torch.tensor([40], dtype=torch.int32, device=DEV)
    good, _ = ops.kv4_attention(q, codes, scales, lens)
    q[0, 2, 77] = bad
    out, lse = ops.kv4_attention(q, codes, scales, lens)
    assert out[0, 2].isnan().all() and lse[0, 2].isnan()
    keep = [0, 1, 3]
    assert torch.equal(out[0, keep], good[0, keep])


def test_attention_of_large_scores(ops):
    """Scores far apart and far from 0: the weights are 0 and 1, none is lost."""
    codes, scales, table = make_cache(1, 1, 64, 200, 16)
    q = 200 * torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(1))
    for kind, t in TYPES.items():
        check_attention(ops, kind, q.to(t), codes, scales, torch.tensor([200], dtype=torch.int32), table=table, weigh=False)
        check_attention(ops, kind, (q * 1e-6).to(t), codes, scales, torch.tensor([200], dtype=torch.int32), table=table)


def test_attention_of_strided_queries(ops):
    """Cut out of a projection, transposed, misaligned, and elements apart."""
    codes, scales, table = on(*make_cache(2, 2, 128, 100, 32))
    lens = torch.tensor([100, 61], dtype=torch.int32, device=DEV)
    x = torch.randn(6, 4, 128, device=DEV).bfloat16()
    want = ops.kv4_attention(x, codes, scales, lens, None, None, table)
    wide = torch.zeros(6, 9, 128, dtype=torch.bfloat16, device=DEV)
    wide[:, 2:6] = x
    flat = torch.zeros(6 * 4 * 128 + 3, dtype=torch.bfloat16, device=DEV)
    odd = flat[3:].view(6, 4, 128)
    odd.copy_(x)
    apart = torch.zeros(6, 4, 128, 2, dtype=torch.bfloat16, device=DEV)
    apart[..., 0] = x
    for y in (wide[:, 2:6], x.transpose(0, 1).contiguous().transpose(0, 1), odd, apart[..., 0]):
        got = ops.kv4_attention(y, codes, scales, lens, None, None, table)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attention_of_nothing(ops):
    codes, scales, table = on(*make_cache(2, 2, 128, 100, 32))
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    out, lse = ops.kv4_attention(torch.zeros(0, 4, 128, device=DEV), codes, scales, lens, None, None, table)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    out, lse = ops.kv4_attention(torch.zeros(0, 4, 128, device=DEV), codes, scales, none)
    assert out.shape == (0, 4, 128)


def test_attention_is_the_same_every_time(ops):
    codes, scales, table = on(*make_cache(3, 2, 128, 3000, 64))
    q = torch.randn(6, 8, 128, device=DEV).bfloat16()
    lens = torch.tensor([3000, 1700, 20], dtype=torch.int32, device=DEV)
    first = ops.kv4_attention(q, codes, scales, lens, None, None, table)
    w = torch.zeros(3, 2, 3000, device=DEV)
    ops.kv4_accumulate(q, first[1], codes, scales, lens, w, None, None, table)
    for _ in range(5):
        again = ops.kv4_attention(q, codes, scales, lens, None, None, table)
        v = torch.zeros_like(w)
        ops.kv4_accumulate(q, again[1], codes, scales, lens, v, None, None, table)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1]) and torch.equal(v, w)


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kind,dim,page", [("bf16", 128, 16), ("bf16", 64, 0), ("f16", 256, 7), ("f32", 128, 0),
                                           ("f32", 64, 64), ("f16", 64, 1)])
def test_append_and_read(ops, kind, dim, page):
    """The new tokens' codes and scales in their places and nowhere else."""
    g = torch.Generator().manual_seed(2)
    new, lens = [3, 0, 40, 1], torch.tensor([10, 5, 70, 1], dtype=torch.int32)
    n, kv = sum(new), 3
    cu = torch.tensor([0] + new).cumsum(0).int()
    x = torch.randn(n, 2 * kv + 1, dim, generator=g) * torch.exp2(torch.randint(-12, 12, (n, 1, 1), generator=g))
    x[0, 0, :32] = 0.0
    x[1, 0, :32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0] * 4)  # on the borders
    x[1, 0, 32:64] = -x[1, 0, :32]
    x[2, 1, :32] = 1e-38 if kind != "f16" else 6e-8
    x = x.to(TYPES[kind])
    codes, scales, table = make_cache(4, kv, dim, 80, page)
    dx, dc, ds, dl, dcu, dt = on(x, codes, scales, lens, cu, table)
    ops.kv4_append(dx[:, :kv], dx[:, kv:2 * kv], dc, ds, dl, dcu, dt)
    want_c, want_s = codes.clone(), scales.clone()
    for plane in (0, 1):
        part = x[:, plane * kv:(plane + 1) * kv].contiguous()
        c, s = ref.quantize(part)
        # the packed form of the same, but for blocks whose scale E8M0 does not
        # have and for quotients of 255 / 1024, the reference's core rounding
        # those to 0.5 (fp8.py:136-140 in bf16) and this one to the nearer 0
        packed_s, packed_c = (t.cpu() for t in ops.quantize_mx_packed(
            (part.float() if kind == "f16" else part).to(DEV), "fp4_e2m1", -1, 32))
        v = torch.ldexp(part.double().unflatten(-1, (-1, 32)), 127 - s.double()[..., None]).to(torch.bfloat16)
        within = (s > 0) & ~(v.abs() == 255 / 1024).any(-1)
        same_c = (packed_c.reshape(n, kv, dim // 32, 16) == c.reshape(n, kv, dim // 32, 16)).all(-1)
        same(packed_s[within], s[within], "packed scales")
        same(same_c[within], torch.ones_like(same_c[within]), "packed codes")
        for b in range(4):
            for k in range(new[b]):
                t = int(lens[b]) - new[b] + k
                _, p, slot = ref.places(table, codes.shape[3], codes.shape[1], b, [t])[0]
                want_c[plane, p, :, slot], want_s[plane, p, :, slot] = c[cu[b] + k], s[cu[b] + k]
    same(dc, want_c, "codes")
    same(ds, want_s, "scales")
    k, v = ops.kv4_read(dc, ds, dl, n, dcu, dt, TYPES[kind])
    for plane, got in ((0, k), (1, v)):
        for b in range(4):
            for i in range(new[b]):
                _, p, slot = ref.places(table, codes.shape[3], codes.shape[1], b, [int(lens[b]) - new[b] + i])[0]
                want = ref.decode(want_c[plane, p, :, slot], want_s[plane, p, :, slot])
                assert torch.equal(got[cu[b] + i].cpu(), want.to(TYPES[kind]))


def test_append_outside(ops):
    """Tokens without a place are not written, read as zeros; blocks with
    an infinity or a NaN are NaN."""
    codes, scales, table = make_cache(3, 1, 64, 32, 16)
    table[1, 0] = -7
    lens = torch.tensor([2, 4, 34], dtype=torch.int32)  # of 4 new ones: 2, 0 and 2 have places
    dc, ds, dl, dt = on(codes, scales, lens, table)
    x = torch.randn(12, 1, 64, device=DEV)
    x[2, 0, 5], x[3, 0, 40] = math.inf, math.nan
    ops.kv4_append(x, x, dc, ds, dl, None, dt)
    k, v = ops.kv4_read(dc, ds, dl, 12, None, dt, torch.float32)
    assert torch.equal(k.nan_to_num(9.0), v.nan_to_num(9.0))
    none = [0, 1, 4, 5, 6, 7, 10, 11]
    assert not k[none].any() and k[[8, 9]].any(-1).all()
    nan = k.isnan()
    assert nan[2, 0, :32].all() and nan[3, 0, 32:].all() and int(nan.sum()) == 64
    changed = ((dc.cpu() != codes).any(-1) | (ds.cpu() != scales).any(-1)).sum()
    assert int(changed) <= 2 * 4


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("lens,budget,recent", [
    ([1, 5, 0, 8], 8, 3), ([100, 64, 65, 63], 64, 16), ([1000, 30, 700, 300], 100, 0), ([1000, 900, 70, 1], 64, 64),
    ([3000, 2999, 1025, 1024], 1023, 7), ([200, 300, 10, 2], 1, 0), ([200, 300, 10, 2], 1, 1)])
@pytest.mark.parametrize("page", [0, 16])
def test_evict(ops, lens, budget, recent, page):
    g = torch.Generator().manual_seed(budget)
    kv, dim, room = 2, 64, max(lens)
    codes, scales, table = make_cache(4, kv, dim, room, page)
    w = torch.rand(4, kv, room, generator=g) ** 4
    w[:, 0] = torch.where(torch.rand(4, room, generator=g) < 0.5, 0.25, w[:, 0])  # many are equal
    w[1, 1, ::7], w[1, 1, 1::7], w[1, 1, 2::7] = -0.0, 0.0, -1.5
    w[0, 1, 0], w[3, 1, 0] = math.nan, math.inf
    lengths = torch.tensor(lens, dtype=torch.int32)
    oc, os_, ot = make_cache(4, kv, dim, budget, 8 if page else 0, 9)
    dc, ds, dt, dw, dl, doc, dos, dot = on(codes, scales, table, w, lengths, oc, os_, ot)
    ow = torch.full((4, kv, budget), 7.0, device=DEV)
    index, kept = ops.kv4_evict(dc, ds, dw, dl, budget, recent, doc, dos, ow, dt, dot)
    want, want_n, want_w = ref.kept(w, lengths, budget, recent)
    same(index, want, "index")
    same(kept, want_n, "lengths")
    same(ow.nan_to_num(-9.0), want_w.nan_to_num(-9.0), "weights")
    want_c, want_s = oc.clone(), os_.clone()
    for b in range(4):
        for h in range(kv):
            for j, t in enumerate(want[b, h].tolist()):
                if t >= 0:
                    _, p, slot = ref.places(table, codes.shape[3], codes.shape[1], b, [t])[0]
                    _, q, at = ref.places(ot, oc.shape[3], oc.shape[1], b, [j])[0]
                    want_c[:, q, h, at], want_s[:, q, h, at] = codes[:, p, h, slot], scales[:, p, h, slot]
    same(doc, want_c, "codes")
    same(dos, want_s, "scales")


@pytest.mark.parametrize("room,budget,recent,kind", [
    (8193, 8192, 0, "random"), (20000, 3000, 500, "random"), (20000, 3000, 500, "few"), (16385, 16000, 1, "equal"),
    (70000, 100, 10, "random"), (150000, 40000, 64, "few"), (150000, 149999, 0, "random"), (30000, 29000, 29000, "few")])
def test_evict_of_long_sequences(ops, room, budget, recent, kind):
    """The selection by slices: the places alone, against a sort."""
    g = torch.Generator().manual_seed(room + budget)
    lens = torch.tensor([room, room - 77, 9000 if room > 9000 else room, min(budget, room), 1, 0], dtype=torch.int32)
    seqs, kv = 6, 2
    codes, scales, table = make_cache(seqs, kv, 64, 16, 0)
    table = torch.zeros(seqs, -(-room // 16), dtype=torch.int32)  # all on one page
    w = torch.randn(seqs, kv, room, generator=g)
    if kind == "few":
        w = (w * 2).round() / 2  # a handful of weights, -0 and 0 among them
    if kind == "equal":
        w.fill_(0.125)
    oc, os_, ot = make_cache(seqs, kv, 64, 16, 0)
    ot = torch.full((seqs, -(-budget // 16)), -1, dtype=torch.int32)
    dc, ds, dt, dw, dl, doc, dos, dot = on(codes, scales, table, w, lens, oc, os_, ot)
    ow = torch.full((seqs, kv, budget), 7.0, device=DEV)
    index, kept = ops.kv4_evict(dc, ds, dw, dl, budget, recent, doc, dos, ow, dt, dot)
    j = torch.arange(room)
    n = lens.long()[:, None, None]
    key = torch.where(j >= n - recent, math.inf, w)
    key = torch.where(j >= n, -math.inf, key)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    want = torch.sort(torch.where(order < n, order, room), dim=-1).values
    live = want < n
    same(index, torch.where(live, want, -1).int(), "index")
    same(kept, lens.clamp(max=budget), "lengths")
    same(ow, torch.where(live, w.gather(-1, want.clamp(max=room - 1)), 0.0), "weights")
    same(doc, oc, "codes")


def test_evict_of_a_token_without_a_page(ops):
    """It is kept as zeros; one that goes to no page is not written."""
    codes, scales, table = make_cache(1, 1, 64, 64, 16)
    table[0, 1] = -1
    oc, os_, ot = make_cache(1, 1, 64, 32, 16, 4)
    ot[0, 1] = oc.shape[1]
    w = torch.zeros(1, 1, 64)
    w[0, 0, 16:32] = 1.0  # the tokens on no page first
    dc, ds, dt, dw, dl, doc, dos, dot = on(codes, scales, table, w, torch.tensor([64], dtype=torch.int32), oc, os_, ot)
    index, _ = ops.kv4_evict(dc, ds, dw, dl, 32, 16, doc, dos, torch.zeros(1, 1, 32, device=DEV), dt, dot)
    assert index[0, 0].tolist() == list(range(16, 32)) + list(range(48, 64))
    p = int(ot[0, 0])
    assert not doc[:, p].any() and not dos[:, p].any()
    doc[:, p], dos[:, p] = oc[:, p].to(DEV), os_[:, p].to(DEV)
    same(doc, oc, "codes")
    same(dos, os_, "scales")


# ---------------------------------------------------------------------------
def test_decode_steps_in_a_graph(ops):
    """A captured step of append, attention and weighing, replayed as the
    sequences grow, against the same steps run eagerly."""
    kv, heads, dim, seqs = 2, 8, 128, 3
    codes, scales, table = make_cache(seqs, kv, dim, 400, 16)
    start = torch.tensor([30, 255, 7], dtype=torch.int32)
    state = [on(codes, scales, table, start) + [torch.zeros(seqs, kv, 400, device=DEV)] for _ in range(2)]
    x = torch.randn(seqs, heads + 2 * kv, dim, device=DEV).bfloat16()

    def step(s):
        c, sc, t, n, w = s
        n.add_(1)
        ops.kv4_append(x[:, heads:heads + kv], x[:, heads + kv:], c, sc, n, None, t)
        out, lse = ops.kv4_attention(x[:, :heads], c, sc, n, None, None, t)
        ops.kv4_accumulate(x[:, :heads], lse, c, sc, n, w, None, None, t)
        return out, lse

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in state[0]])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(state[0])
    for i in range(6):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)))
        want = step(state[1])
        torch.cuda.synchronize()
        graph.replay()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
        for a, b in zip(state[0], state[1]):
            assert torch.equal(a, b)


def test_on_another_stream(ops):
    codes, scales, table = on(*make_cache(2, 2, 128, 500, 16))
    q = torch.randn(2, 8, 128, device=DEV).bfloat16()
    lens = torch.tensor([500, 300], dtype=torch.int32, device=DEV)
    want = ops.kv4_attention(q, codes, scales, lens, None, None, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.kv4_attention(q, codes, scales, lens, None, None, table)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_the_serving_example(vqx):
    """Its steps together: the attention is as near as 4 bits let it be, the
    budget is kept, and the weights of a decode step are those of its heads."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_kv4.py")
    spec = importlib.util.spec_from_file_location("serve_kv4", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    seqs, budget, steps, heads = 3, 96, 5, 16
    r = example.serve(seqs=seqs, prompt=300, budget=budget, steps=steps, heads=heads, width=256, recent=16)
    assert r["kept"] == [budget + steps] * seqs
    # a value of 4 bits is off by at most a quarter of itself, or of 0.5 steps
    # below its block's least level; the attention averages many
    assert 0 < r["error"] < 0.25
    assert r["outputs"].isfinite().all()
    index = r["index"]
    assert bool((index[..., 1:] > index[..., :-1]).all()) and bool((index >= 0).all())
    # each step adds 1 for each query head: 16 admission queries and 5 steps, of
    # which eviction kept a part
    total = r["weights"].sum((1, 2)).cpu()
    assert bool((total <= heads * (16 + steps) * (1 + 2.0 ** -10)).all())
    assert bool((total >= heads * steps * (1 - 2.0 ** -10)).all())


@pytest.mark.parametrize("many", [False, True])
def test_a_cache_past_32_bits(ops, many):
    """The same pages at the far end of a cache of 5 GiB a plane: every operator
    finds them there and writes nothing else."""
    dim, kv, page, seqs = 128, 2, 64, 2
    pages = 5 * 2 ** 30 // (kv * page * dim // 2)
    far = torch.tensor([[pages - 1, pages - 3], [pages - 2, pages - 5]], dtype=torch.int32, device=DEV)
    near_table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    if many:  # the kernel for many rows, by room
        far, near_table = (torch.nn.functional.pad(t, (0, 4000), value=-1) for t in (far, near_table))
    big_c = torch.empty(2, pages, kv, page, dim // 2, dtype=torch.uint8, device=DEV)
    big_s = torch.empty(2, pages, kv, page, dim // 32, dtype=torch.uint8, device=DEV)
    c, s, _ = on(*make_cache(4, kv, dim, page, 0))
    big_c[:, far[:, :2].flatten().long()], big_s[:, far[:, :2].flatten().long()] = c, s
    lens = torch.tensor([128, 100], dtype=torch.int32, device=DEV)
    new = 40 if many else 1
    x = torch.randn(seqs * new, 8, dim, device=DEV).bfloat16()
    got = []
    for codes, scales, table in ((big_c, big_s, far), (c, s, near_table)):
        ops.kv4_append(x[:, 4:6], x[:, 6:], codes, scales, lens, None, table)
        k, v = ops.kv4_read(codes, scales, lens, seqs * new, None, table)
        out, lse = ops.kv4_attention(x[:, :4], codes, scales, lens, None, None, table)
        w = torch.zeros(seqs, kv, 128, device=DEV)
        ops.kv4_accumulate(x[:, :4], lse, codes, scales, lens, w, None, None, table)
        oc, os_, ow = torch.zeros(2, 2, kv, 50, 64, dtype=torch.uint8, device=DEV), torch.zeros(
            2, 2, kv, 50, 4, dtype=torch.uint8, device=DEV), torch.zeros(seqs, kv, 50, device=DEV)
        index, _ = ops.kv4_evict(codes, scales, w, lens, 50, 8, oc, os_, ow, table)
        got.append((k, v, out, lse, w, index, oc, os_, ow))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    # and into it
    ops.kv4_evict(c, s, w, lens, 50, 8, big_c, big_s, ow, near_table, far[:, :2].contiguous())
    for b in range(seqs):
        same(big_c[:, int(far[b, 0]), :, :50], oc[:, b], "codes")
        same(big_s[:, int(far[b, 0]), :, :50], os_[:, b], "scales")
