"""The 4-bit cache's operators where results go wrong first: places that count
nothing and hold anything, values far apart in size, rows without tokens."""

import pytest
import torch

from tests.test_gpu_kv4 import TYPES, check_attention, make_cache, ops  # noqa: F401

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
