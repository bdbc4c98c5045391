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
