"""Packed forms whose codes and scales are both strided views."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale_dtype", [torch.uint8, torch.float32])
@pytest.mark.parametrize("rows", [64, 4096])
def test_dequantize_of_strided_codes_and_scales(vqx, rows, scale_dtype):
    """Both are copied; neither copy may take the other's memory before the
    kernel has read it."""
    g = torch.Generator().manual_seed(rows)
    codes = torch.randint(0, 256, (rows, 64), generator=g, dtype=torch.uint8).cuda()
    scale = torch.randint(120, 130, (rows, 4), generator=g, dtype=torch.uint8).cuda()
    if scale_dtype == torch.float32:
        scale = torch.exp2(scale.float() - 127)
    take = lambda c, s: torch.ops.quantized_ops.dequantize_mx_packed(  # noqa: E731
        c, s, "fp4_e2m1", 32, [rows, 128], torch.bfloat16)
    want = take(codes, scale)
    wide_codes, wide_scale = torch.zeros(rows, 128, dtype=torch.uint8).cuda(), torch.zeros(rows, 8).to(scale_dtype).cuda()
    wide_codes[:, ::2], wide_scale[:, ::2] = codes, scale
    torch.cuda.synchronize()
    for _ in range(3):
        assert torch.equal(take(wide_codes[:, ::2], wide_scale[:, ::2]), want)
