"""Rotary positions for queries and keys.

``torch.ops.quantized_ops.rotary`` and ``rotary_frequencies``, this package's
own: what a decoder does to its queries and keys before ``kv4_append`` and
``kv4_attention``.  ``kv4_append_rotary`` (``kv4.py``) does it on the way into
the cache; this one stands alone, and gradients pass through it.
"""

import math

import torch
from torch._functorch.autograd_function import enable_single_level_autograd_function
from torch.autograd import forward_ad
from torch.autograd.function import _SingleLevelFunction

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
    gradient of x is the turn back, a tangent's the turn; positions and freqs have
    none.  torch.func's transforms take it too (vmap one element at a time)."""
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


_keys = torch._C._dispatch_keys
_PLAIN = torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA)
for _k in ("ADInplaceOrView", "AutogradCUDA", "AutocastCUDA"):
    _PLAIN = _PLAIN | torch._C.DispatchKeySet(getattr(torch._C.DispatchKey, _k))


def _plain(x, positions, freqs):
    """Whether all that the dispatcher would do below autograd is to call the kernel:
    there is no mode, and no tensor is of a kind that has a say before its data is
    read, as a transform's, a tracer's or a negative view (a second way through the
    dispatcher is 3 us of a call's 11, and 10 in a backward pass, whose thread has
    just been woken; looking at the keys is 1)."""
    return (_keys(x) == _PLAIN and _keys(freqs) == _PLAIN and _keys(positions) == _PLAIN
            and not torch._C._len_torch_dispatch_stack())


def _below(x, positions, freqs, interleaved, factor, back):
    """The turn below autograd, by the dispatcher."""
    with torch._C._AutoDispatchBelowAutograd():
        return torch.ops.quantized_ops.rotary(x, positions, freqs, interleaved=interleaved, factor=factor, back=back)


class _Rotary(_SingleLevelFunction):
    """The turn with the turn back, its transpose, as gradient, and a tangent's turn
    as tangent.  Like any of autograd's kernels it is for one level of it: torch.func's
    transforms come here level by level.  modes: None where the kernel may be called
    at once, or whether gradients and tangents are wanted, which those below are to
    know."""

    @staticmethod
    def forward(ctx, x, positions, freqs, interleaved, factor, back, modes):
        ctx.save_for_backward(positions, freqs)
        ctx.how = interleaved, factor, back
        if modes is None:
            return rotary(x, positions, freqs, interleaved=interleaved, factor=factor, back=back)
        ctx.save_for_forward(positions, freqs)
        with torch.set_grad_enabled(modes[0]), forward_ad._set_fwd_grad_enabled(modes[1]):
            return _below(x, positions, freqs, interleaved, factor, back)

    @staticmethod
    def backward(ctx, grad):
        positions, freqs = ctx.saved_tensors
        interleaved, factor, back = ctx.how
        at_once = not torch.is_grad_enabled() and _plain(grad, positions, freqs)
        turn = rotary if at_once else torch.ops.quantized_ops.rotary
        return turn(grad, positions, freqs, interleaved=interleaved, factor=factor, back=not back), *[None] * 6

    @staticmethod
    def jvp(ctx, tangent, *_):
        positions, freqs = ctx.saved_tensors
        interleaved, factor, back = ctx.how
        return torch.ops.quantized_ops.rotary(tangent, positions, freqs, interleaved=interleaved, factor=factor, back=back)


@torch.library.impl(quantized_ops_lib, "rotary", "Autograd")
def _rotary_autograd(x, positions, freqs, *, interleaved=False, factor=1.0, back=False):
    grads, tangents = torch.is_grad_enabled(), forward_ad._current_level >= 0
    if (grads and freqs.requires_grad) or (tangents and forward_ad.unpack_dual(freqs).tangent is not None):
        kv4._refuse("rotary", "freqs have no gradient here")
    if not tangents and _plain(x, positions, freqs):
        if grads and x.requires_grad:
            return _Rotary.apply(x, positions, freqs, interleaved, factor, back, None)
        return rotary(x, positions, freqs, interleaved=interleaved, factor=factor, back=back)
    if tangents or (grads and x.requires_grad):
        with enable_single_level_autograd_function():
            return _Rotary.apply(x, positions, freqs, interleaved, factor, back, (grads, torch._C._is_fwd_grad_enabled()))
    return _below(x, positions, freqs, interleaved, factor, back)


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
