"""Which kernel the 4-bit cache's attention runs, and how near each comes."""

import pytest
import torch
from torch.profiler import ProfilerActivity, profile

from tests import kv4_reference as ref
from tests import test_gpu_kv4 as base
from tests.test_gpu_kv4 import TYPES, make_cache, near, on, ops, widened  # noqa: F401

pytestmark = pytest.mark.gpu


def kernels_of(call):
    """What a call returns, and the names of the cache's kernels that it ran."""
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        result = call()
        torch.cuda.synchronize()
    names = " ".join(e.name for e in p.events())
    if "_kernel" not in names:
        pytest.skip("the profiler sees no kernels here")
    return result, {n for n in ("rows", "block", "join", "weigh") if f"kv4_{n}_kernel" in names}


@pytest.mark.parametrize("i", range(len(base.MANY)))
def test_small_tests_reach_the_kernel_for_many_rows(ops, i, monkeypatch):  # noqa: F811
    """And with weights of two bf16 terms, the second rounded to half a step:
    off by 2^-8 of 2^-8 of themselves."""
    monkeypatch.setitem(base.WEIGHT, "bf16", 2.0 ** -16)
    _, found = kernels_of(lambda: base.test_attention_many_rows(ops, i))
    assert "block" in found and "rows" not in found


@pytest.mark.parametrize("i", [i for i, c in enumerate(base.CASES) if c[0] == "bf16"])
def test_small_calls_run_the_kernel_for_few_rows(ops, i, monkeypatch):  # noqa: F811
    monkeypatch.setitem(base.WEIGHT, "bf16", 2.0 ** -16)
    _, found = kernels_of(lambda: base.test_attention(ops, i))
    assert "rows" in found and "block" not in found


@pytest.mark.parametrize("kind,dim,page", [("bf16", 128, 16), ("f16", 64, 64), ("f32", 256, 0)])
def test_many_rows_ragged_and_more_than_most(ops, kind, dim, page):  # noqa: F811
    """The kernel for many rows with sequences of none, one and many new tokens,
    some of them more than `most`: those rows are NaN, the others as they were."""
    new, most = [0, 1, 170, 9, 150, 130], 100
    lens = torch.tensor([40, 300, 170, 4, 260, 140], dtype=torch.int32)
    cu = torch.tensor([0] + new).cumsum(0).int()
    codes, scales, table = widened(*make_cache(6, 2, dim, 300, page), 100)
    q = torch.randn(sum(new), 6, dim, generator=torch.Generator().manual_seed(3)).to(TYPES[kind])
    _, found = kernels_of(lambda: base.check_attention(ops, kind, q, codes, scales, lens, cu, max(new), table, weigh=False))
    assert "block" in found and "rows" not in found
    d = on(q, codes, scales, lens, cu, table)
    want, want_lse = ops.kv4_attention(d[0], d[1], d[2], d[3], d[4], max(new), d[5])
    (out, lse), found = kernels_of(lambda: ops.kv4_attention(d[0], d[1], d[2], d[3], d[4], most, d[5]))
    assert "block" in found and "rows" not in found
    beyond = torch.cat([torch.arange(n) >= most for n in new])
    assert out[beyond].isnan().all() and lse[beyond].isnan().all()
    # the same sums, cut into other splits
    off = torch.finfo(TYPES[kind]).eps + 2.0 ** -15
    near(out[~beyond], want[~beyond].cpu().double(), off * 8, "out")
    near(lse[~beyond], want_lse[~beyond].cpu().double(), 2.0 ** -16, "lse")


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("many", [False, True])
def test_the_norm_of_the_error(ops, kind, many):  # noqa: F811
    """Little more than that of rounding the right result: weights of two bf16
    terms (2^-16) add less than 0.1% to it, of one term (2^-8) some 40%."""
    new, length = (64, 2000) if many else (8, 2000)
    codes, scales, table = make_cache(1, 1, 128, length, 64)
    if many:
        codes, scales, table = widened(codes, scales, table, 8)
    q = torch.randn(new, 2, 128, generator=torch.Generator().manual_seed(1)).to(TYPES[kind])
    lens = torch.tensor([length], dtype=torch.int32)
    d = on(q, codes, scales, lens, table)
    (out, _), found = kernels_of(lambda: ops.kv4_attention(d[0], d[1], d[2], d[3], None, None, d[4]))
    assert ("block" if many else "rows") in found
    want = ref.attention(q, codes, scales, lens, None, table)[0]
    off, rounding = (out.cpu().double() - want).norm(), (want.to(TYPES[kind]).double() - want).norm()
    assert float(off) <= 1.02 * float(rounding), (float(off / want.norm()), float(rounding / want.norm()))
