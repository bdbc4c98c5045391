"""How a tree's weights are held: two bf16 terms each (fp32: three), in the kernel for
few rows and in the one for many.  With one term, which the tolerance here tells from
two, outputs of values that cancel would lose half of their digits."""

import pytest
import torch

from tests.test_gpu_kv4 import near, on
from tests.test_gpu_kv4_pages import forest, signed
from tests.test_gpu_kv4_tree import attention, scene
from tests.test_gpu_kv4_tree_windows import tolerances

DEV = "cuda"
# few rows; almost all of the workgroups' rows, over 16 kv heads of 8 query heads
SHAPES = {"few": (2, 4, [200, 31, 700], [12, 1, 30]),
          "many": (16, 8, [100, 64, 200, 90, 65, 150, 71, 480], [64, 64, 60, 64, 57, 64, 64, 64])}
KINDS = [("bf16", 64), ("bf16", 128), ("bf16", 256), ("f16", 64), ("f16", 128), ("f16", 256), ("f32", 128)]


def make(kind, dim, shape):
    kv, group, lengths, news = SHAPES[shape]
    q, codes, scales, lens, cu, table = scene(kind, dim, kv, group, lengths, news, 16, 5)
    return (q, codes, scales, lens), forest(news, 3)[0], cu, table


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dim", KINDS)
@pytest.mark.parametrize("shape", list(SHAPES))
def test_weights(vqx, kind, dim, shape):
    inputs, tree, cu, table = make(kind, dim, shape)
    dev = on(*inputs, torch.tensor([signed(m) for m in tree]), cu)
    out, lse = torch.ops.quantized_ops.kv4_tree_attention(*dev, 64, table.to(DEV))
    want = attention(*inputs, tree, cu, table)
    tol, lse_tol = tolerances(inputs[0], kind, *want)
    near(out, want[0], tol, "out")
    near(lse, want[1], lse_tol, "lse")


@pytest.mark.parametrize("kind,dim", KINDS)
def test_one_term_would_be_seen(monkeypatch, kind, dim):
    """The same form with its weights rounded to bf16 once lies outside."""
    inputs, tree, cu, table = make(kind, dim, "few")
    want = attention(*inputs, tree, cu, table)
    tol, _ = tolerances(inputs[0], kind, *want)
    exp = torch.exp
    monkeypatch.setattr(torch, "exp", lambda x: exp(x).bfloat16().double())
    lost = attention(*inputs, tree, cu, table)[0]
    assert bool(((lost - want[0]).abs() > tol).any())  # one element is enough for the test above to fail
    assert bool(((want[0].to(inputs[0].dtype).double() - want[0]).abs() <= tol).all())
