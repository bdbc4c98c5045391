"""Attention of drafted tokens within windows that are cut into several splits, also
where a sequence has more new tokens than the call was told of."""

import pytest
import torch

from tests.test_gpu_kv4 import near, on, same
from tests.test_gpu_kv4_pages import forest, signed
from tests.test_gpu_kv4_tree import attention, scene

pytestmark = pytest.mark.gpu

DEV = "cuda"
# A weight is held as two bf16 terms, each to half a step of what is left: 2^-18
# of it (fp32: three, 2^-27).
WEIGHT = {"bf16": 2.0 ** -18, "f16": 2.0 ** -18, "f32": 2.0 ** -27}


@pytest.fixture(scope="module")
def ops(vqx):
    return torch.ops.quantized_ops


def tolerances(q, kind, w_out, w_lse, mass, err):
    """Of the outputs: twice a score's error on a weight and its sum, sums of fp32 in
    some order, the weights' terms, the output's half step.  Of lse: the score's
    error, sums and logarithm of fp32."""
    rel = 2 * err + 64 * 2.0 ** -24
    tol = torch.finfo(q.dtype).eps / 2 * w_out.abs() + (rel[..., None] + WEIGHT[kind]) * (1 + 2.0 ** -8) * mass + 1e-30
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half of its smallest subnormal
    return tol, err + 64 * 2.0 ** -24 + 8 * 2.0 ** -24 * w_lse.abs().nan_to_num(0, 0, 0)


# kind, dim, kv, group, lengths, new tokens, most, window, page, slopes
WINDOWS = [
    ("bf16", 64, 2, 4, [10000, 4100], [12, 40], 40, 1950, 64, False),
    ("f16", 128, 1, 2, [9000, 700], [64, 5], 64, 4000, 0, True),
    ("f32", 64, 1, 1, [70000], [7], 7, 66000, 128, False),  # more splits than a wave joins
    ("f32", 256, 1, 1, [6000, 5000, 1], [3, 20, 1], 20, 2500, 48, False),
    ("bf16", 64, 4, 8, [26000], [64], 64, 24900, 128, False),  # the kernel for many rows
]
BEYOND = [
    ("bf16", 64, 1, 1, [5000], [3000], 64, 1990, 0, False),
    ("f32", 64, 2, 2, [10000, 10000], [64, 64], 8, 1976, 64, False),
    ("f16", 128, 2, 1, [10000, 9000], [200, 130], 16, 4000, 16, True),
    ("bf16", 128, 1, 4, [9000, 300, 8000], [128, 3, 64], 64, 1920, 64, False),
    ("bf16", 64, 4, 8, [26000], [100], 64, 24900, 128, False),
]


@pytest.mark.parametrize("kind,dim,kv,group,lengths,news,most,window,page,sloped", WINDOWS + BEYOND)
def test_windows_in_splits(ops, kind, dim, kv, group, lengths, news, most, window, page, sloped):
    """Rows up to `most` against the 64-bit form of a sequence that has no more;
    those beyond are NaN."""
    q, codes, scales, lens, cu, table = scene(kind, dim, kv, group, lengths, news, page, 1)
    slopes = torch.linspace(0.0001, 0.002, kv * group) if sloped else None
    there = [min(c, most) for c in news]
    rows, tree = [], []
    for b, masks in enumerate(there):
        tree += forest([masks], b)[0] + [0] * (news[b] - masks)
        rows += range(int(cu[b]), int(cu[b]) + masks)
    dev = on(q, codes, scales, lens, torch.tensor([signed(m) for m in tree]), cu)
    out, lse = ops.kv4_tree_attention(*dev, most, *on(table), window=window, slopes=None if slopes is None else slopes.to(DEV))
    torch.cuda.synchronize()
    want = attention(q[rows], codes, scales, lens - torch.tensor(news) + torch.tensor(there), [tree[i] for i in rows],
                     torch.tensor([0] + there).cumsum(0), table, window=window, slopes=slopes)
    tol, lse_tol = tolerances(q, kind, *want)
    near(out[rows], want[0], tol, "out")
    near(lse[rows], want[1], lse_tol, "lse")
    beyond = sorted(set(range(q.shape[0])) - set(rows))
    assert bool(out[beyond].isnan().all()) and bool(lse[beyond].isnan().all())


@pytest.mark.parametrize("kind,dim,kv,group,lengths,news,most,window,page,sloped", BEYOND)
def test_bits_beyond_the_most(ops, kind, dim, kv, group, lengths, news, most, window, page, sloped):
    """They do not count."""
    q, codes, scales, lens, cu, table = on(*scene(kind, dim, kv, group, lengths, news, page, 2))
    some = torch.randint(-2 ** 62, 2 ** 62, (sum(news),), generator=torch.Generator().manual_seed(3)).to(DEV)
    known = (1 << most) - 1 if most < 64 else -1
    one, two = (ops.kv4_tree_attention(q, codes, scales, lens, t, cu, most, table, window=window)
                for t in (some & known, some | ~known))
    for a, b, name in zip(one, two, ("out", "lse")):
        assert torch.equal(a.isnan(), b.isnan()), name
        same(a.nan_to_num(7.0), b.nan_to_num(7.0).cpu(), name)
