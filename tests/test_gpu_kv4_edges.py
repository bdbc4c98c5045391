"""The 4-bit cache's operators where results go wrong first: places that count
nothing and hold anything, values far apart in size, rows without tokens."""

import pytest
import torch

from tests import kv4_reference as ref
from tests.test_gpu_kv4 import TYPES, check_attention, make_cache, near, on, ops, widened  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,dim", [("bf16", 128), ("f16", 64), ("f32", 256)])
@pytest.mark.parametrize("lens,new,group,how", [
    ([6], 10, 1, {}), ([1], 2, 4, {}), ([3, 40], 19, 1, {}), ([17, 0, 5], 20, 2, dict(window=4)),
    ([1, 2], 33, 1, dict(softcap=5.0)), ([30], 31, 3, dict(slopes=True))])
def test_more_new_tokens_than_tokens(ops, kind, dim, lens, new, group, how):
    """Sequences shorter than their new tokens: the first rows stand before the
    beginning and see nothing, the others are weighed like any."""
    kv, seqs = 2, len(lens)
    codes, scales, table = make_cache(seqs, kv, dim, max(lens), 16)
    g = torch.Generator().manual_seed(new)
    q = torch.randn(seqs * new, kv * group, dim, generator=g).to(TYPES[kind])
    how = dict(how)
    if how.get("slopes"):
        how["slopes"] = torch.exp2(-8.0 * torch.arange(1, kv * group + 1) / (kv * group))
    check_attention(ops, kind, q, codes, scales, torch.tensor(lens, dtype=torch.int32), table=table, **how)


def value_byte(codes, scales, table, b, t, byte, block=None, code=None):
    """Sets the scale byte of token t's values, of one block or of all."""
    _, p, slot = ref.places(table, codes.shape[3], codes.shape[1], b, [t])[0]
    at = slice(None) if block is None else block
    scales[1, p, :, slot, at] = byte
    if code is not None:
        codes[1, p, :, slot] = code | code << 4


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 0)])
@pytest.mark.parametrize("many", [False, True])
def test_values_of_any_size(ops, kind, dim, page, many):
    """A block of a head 2^60 above its neighbour, and single tokens 2^70 above
    the others: rows that do not see them, and the other block, lose nothing."""
    codes, scales, table = make_cache(2, 1, dim, 200, page)
    scales[1, ..., -1] += 60
    for b, t, byte in ((0, 190, 197), (0, 40, 20), (1, 90, 197)):
        value_byte(codes, scales, table, b, t, byte, 0)
    if many:
        codes, scales, table = widened(codes, scales, table, 2 * 8)
    q = torch.randn(2 * 40, 3, dim, generator=torch.Generator().manual_seed(1)).to(TYPES[kind])
    check_attention(ops, kind, q, codes, scales, torch.tensor([200, 100], dtype=torch.int32), table=table, weigh=False)


@pytest.mark.parametrize("many", [False, True])
def test_values_of_the_smallest_size(ops, many):
    """Positive values near 2^-120, some of them in blocks of the smallest scale."""
    codes, scales, table = make_cache(1, 1, 128, 100, 16)
    codes &= 0x77
    scales[1] = torch.randint(0, 6, scales[1].shape, generator=torch.Generator().manual_seed(2))
    if many:
        codes, scales, table = widened(codes, scales, table, 8)
    q = torch.randn(40, 3, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    lens = torch.tensor([100], dtype=torch.int32)
    d = on(q, codes, scales, lens, table)
    out, _ = ops.kv4_attention(d[0], d[1], d[2], d[3], None, None, d[4])
    want = ref.attention(q, codes, scales, lens, None, table)[0]
    # all of one sign: the output's half step, the weights' 2^-8 at most, and
    # the spacing of bf16 below its normal range
    near(out, want, 2.0 ** -7 * want + 2.0 ** -133, "out")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [8, 64])
@pytest.mark.parametrize("many", [False, True])
def test_tokens_without_a_page_over_any_bytes(ops, kind, dim, page, many):
    """The first row of the cache, which stands in for a token without a page,
    holds values past every type's range: nothing of it is seen."""
    codes, scales, table = make_cache(2, 1, dim, 160, page)
    codes, scales = (torch.cat([x[:, :1], x], 1) for x in (codes, scales))
    table = table + 1
    codes[:, 0], scales[:, 0] = 0xFF, 254
    table[0, 1], table[1, 0], table[1, -1] = -1, codes.shape[1], 2 ** 31 - 1
    new = 20 if many else 1
    if many:
        codes, scales, table = widened(codes, scales, table, 2 * -(-new * 3 // 16))
    q = torch.randn(2 * new, 3, dim, generator=torch.Generator().manual_seed(1)).to(TYPES[kind])
    check_attention(ops, kind, q, codes, scales, torch.tensor([160, 150], dtype=torch.int32), table=table)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [8, 64])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("byte,code", [(253, 6), (254, 4), (254, 15)])
def test_values_past_the_range_in_masked_places(ops, kind, dim, page, many, byte, code):
    """Values of 2^128 and of -1.5 * 2^129: rows that do not see them are as they
    were; rows that do have their share of them, where the type holds it."""
    new, lens = 30, torch.tensor([130, 96], dtype=torch.int32)
    codes, scales, table = make_cache(2, 1, dim, 160, page)
    if many:
        codes, scales, table = widened(codes, scales, table, 2 * -(-new * 3 // 16))
    q = torch.randn(2 * new, 3, dim, generator=torch.Generator().manual_seed(1)).to(TYPES[kind])
    d = on(q, codes, scales, lens, table)
    before, _ = ops.kv4_attention(d[0], d[1], d[2], d[3], None, None, d[4])
    value_byte(codes, scales, table, 0, 125, byte, code=code)
    dc, ds = on(codes, scales)
    out, lse = ops.kv4_attention(d[0], dc, ds, d[3], None, None, d[4])
    sees = torch.zeros(2 * new, dtype=torch.bool)
    sees[25:30] = True
    assert torch.equal(out[~sees], before[~sees])
    want = ref.attention(q, codes, scales, lens, None, table)[0][sees]
    top = torch.finfo(TYPES[kind]).max
    got, held = out[sees].cpu().double(), want.abs() < 0.99 * top
    # one value outweighs all others: its own weight's error, the half step
    off = (got - want).abs() / want.abs()
    assert not got.isnan().any() and float(off[held].max() if held.any() else 0.0) <= 2.0 ** -7
    past = want.abs() > 1.01 * top
    assert bool(got[past].isinf().all()) and torch.equal(got[past].sign(), want[past].sign())
    assert held.any() or kind == "f16"


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("new,length", [(1, 40), (1, 9000), (40, 200), (300, 900)])
def test_a_mean_of_the_largest_values(ops, kind, new, length):
    """Values of 2^127 each: their sum is past the range, their mean is not."""
    codes, scales, table = make_cache(1, 2, 128, length, 64)
    codes[1], scales[1] = 0x44, 253
    q = torch.randn(new, 8, 128, generator=torch.Generator().manual_seed(1)).to(TYPES[kind])
    d = on(q, codes, scales, torch.tensor([length], dtype=torch.int32), table)
    out, _ = ops.kv4_attention(d[0], d[1], d[2], d[3], None, None, d[4])
    want = torch.full(out.shape, 2.0 ** 127, dtype=torch.float64)
    # weights and their sum, each off by its terms and by fp32's sums
    near(out, want, (torch.finfo(TYPES[kind]).eps / 2 + (2.0 ** -16 if kind == "bf16" else 0) + 2.0 ** -19) * want, "out")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.0, 2.0 ** -110, -2.0 ** -110])
def test_scales_of_next_to_nothing(ops, kind, many, scale):
    """Keys of 2^105: a scale of 0 makes every score 0, one of 2^-110 makes
    ordinary scores of them."""
    codes, scales, table = make_cache(2, 1, 128, 100, 16)
    scales[0] += 105
    if many:
        codes, scales, table = widened(codes, scales, table, 2 * 8)
    new = 40 if many else 1
    q = torch.randn(2 * new, 3, 128, generator=torch.Generator().manual_seed(1)).to(TYPES[kind])
    lens = torch.tensor([100, 77], dtype=torch.int32)
    check_attention(ops, kind, q, codes, scales, lens, table=table, scale=scale)
    check_attention(ops, kind, q, codes, scales, lens, table=table, scale=scale, softcap=3.0)


@pytest.mark.parametrize("how", [dict(window=20), dict(slopes=True), dict(window=33, slopes=True, softcap=5.0)])
def test_distances_in_an_evicted_cache(ops, how):
    """Windows and slopes count the slots of the cache that eviction has filled."""
    seqs, kv, group, dim, budget = 2, 2, 3, 64, 48
    codes, scales, table = make_cache(seqs, kv, dim, 200, 16)
    oc, os_, ot = make_cache(seqs, kv, dim, budget, 8, 9)
    w = torch.rand(seqs, kv, 200, generator=torch.Generator().manual_seed(1))
    lens = torch.tensor([200, 30], dtype=torch.int32)
    d = on(codes, scales, w, lens, oc, os_, torch.zeros(seqs, kv, budget), table, ot)
    _, kept = ops.kv4_evict(d[0], d[1], d[2], d[3], budget, 8, d[4], d[5], d[6], d[7], d[8])
    how = dict(how)
    if how.get("slopes"):
        how["slopes"] = torch.exp2(-8.0 * torch.arange(1, kv * group + 1) / (kv * group))
    q = torch.randn(seqs, kv * group, dim, generator=torch.Generator().manual_seed(2)).bfloat16()
    check_attention(ops, "bf16", q, d[4].cpu(), d[5].cpu(), kept.cpu(), table=ot, **how)


@pytest.mark.parametrize("kind,dim,length,new", [("bf16", 64, 100001, 1), ("f32", 128, 70000, 2), ("f16", 256, 18000, 1)])
def test_more_splits_than_lanes(ops, kind, dim, length, new):
    """One head of one long sequence, cut into up to a hundred splits; the last
    part of it weighs most, as a slope has it, or all of it the same."""
    codes, scales, table = make_cache(1, 1, dim, length, 64)
    q = torch.randn(new, 2, dim, generator=torch.Generator().manual_seed(1)).to(TYPES[kind])
    lens = torch.tensor([length], dtype=torch.int32)
    check_attention(ops, kind, q, codes, scales, lens, table=table, scale=0.01)
    check_attention(ops, kind, q, codes, scales, lens, table=table, slopes=torch.tensor([0.001, 0.5]))
