"""Rotary positions for queries and keys.

``torch.ops.quantized_ops.rotary`` and ``rotary_frequencies``, this package's
own: what a decoder does to its queries and keys before ``kv4_append`` and
``kv4_attention``.  ``kv4_append_rotary`` (``kv4.py``) does it on the way into
the cache; this one stands alone, and gradients pass through it.
"""

import math

import torch

from .. import _lib
from . import kv4
from .quantized import quantized_ops_lib

quantized_ops_lib.define(
    "rotary(Tensor x, Tensor positions, Tensor freqs, *, bool interleaved=False, float factor=1.0, "
    "bool back=False) -> Tensor")


@torch.library.impl(quantized_ops_lib, "rotary", "CUDA")
def rotary(x, positions, freqs, *, interleaved=False, factor=1.0, back=False):
    """x [n, heads, D] (D a multiple of 8 up to 1024) with the first 2 len(freqs)
    elements of each head turned: pair i, (x[i], x[i + len(freqs)]) or
    (interleaved) (x[2 i], x[2 i + 1]), by the angle positions[token] * freqs[i]
    and times factor; back: by the negative angle.  positions: int32 [n]; freqs:
    fp32.  Angles and products are in 64 bits, rounded once to x's dtype.  The
    gradient of x is the turn back; positions and freqs have none."""
    what = "rotary"
    _lib.require_device(x, what)
    device = x.device
    if x.dim() != 3 or x.shape[2] % 8 or not 8 <= x.shape[2] <= 1024:
        kv4._refuse(what, f"x must be [tokens, heads, D] with D a multiple of 8 up to 1024, not {list(x.shape)}")
    n, heads, dim = x.shape
    t = kv4._turn(freqs, positions, n, dim, interleaved, factor, back, what, device)
    x, sn, sh, tag = kv4._rows(x, None, dim, "x", what, device)
    out = x.new_empty((n, heads, dim))
    kv4._launch("vqx_rotary", x, x.data_ptr(), tag, n, heads, dim, sn, sh, t, out.data_ptr())
    return out


@torch.library.register_fake("quantized_ops::rotary")
def _(x, positions, freqs, *, interleaved=False, factor=1.0, back=False):
    return x.new_empty(x.shape)


def _save(ctx, inputs, keyword_only_inputs, output):
    _, positions, freqs = inputs
    if freqs.requires_grad:
        raise ValueError("vqx: rotary: freqs have no gradient here")
    ctx.save_for_backward(positions, freqs)
    ctx.how = keyword_only_inputs


def _back(ctx, grad):
    positions, freqs = ctx.saved_tensors
    how = ctx.how
    # a turn's transpose is the turn back
    return torch.ops.quantized_ops.rotary(grad, positions, freqs, interleaved=how["interleaved"], factor=how["factor"],
                                          back=not how["back"]), None, None


torch.library.register_autograd("quantized_ops::rotary", _back, setup_context=_save)


def rotary_frequencies(turned, base=10000.0, *, stretch=1.0, trained=None, slow=1.0, fast=4.0, device=None):
    """fp32 [turned / 2]: base ** (-2 i / turned) radians from one position to
    the next.  For a context `stretch` times as long as the model's own: without
    `trained` every frequency is divided by stretch; with it (the positions that
    the model was trained on) only those that make fewer than `slow` whole turns
    within them, those with more than `fast` stay, and between the two it goes
    linearly with the turns."""
    if turned < 2 or turned % 2:
        raise ValueError(f"vqx: rotary_frequencies: an even number of turned elements, not {turned}")
    if not (base > 0 and stretch > 0 and (trained is None or trained > 0) and 0 <= slow < fast):
        raise ValueError("vqx: rotary_frequencies: base, stretch and trained are positive, slow is below fast")
    f = base ** (-torch.arange(0, turned, 2, dtype=torch.float64) / turned)
    if trained is None:
        f = f / stretch
    else:
        keep = ((trained * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f * keep + f / stretch * (1 - keep)
    return f.float().to(device)
