"""Tokens drawn from logits.

``torch.ops.quantized_ops.sample_tokens``, this package's own: the end of a decode
step, and what ``kv4_accept`` compares drafted tokens with.  No gradient passes
through it.
"""

import ctypes

import torch

from .. import _lib
from . import kv4
from .quantized import quantized_ops_lib

quantized_ops_lib.define(
    "sample_tokens(Tensor logits, Tensor random, Tensor? temperature=None, Tensor? top_k=None, Tensor? top_p=None, "
    "Tensor? min_p=None) -> (Tensor, Tensor)")


def _of_rows(t, rows, dtype, name, what, device):
    """The address of t, one value a row, or None."""
    if t is None:
        return None
    if t.dtype != dtype or t.shape != (rows,) or not t.is_contiguous():
        kv4._refuse(what, f"{name} must be a contiguous {dtype} tensor of shape [{rows}], not {t.dtype} {list(t.shape)}")
    if t.device != device:
        kv4._refuse(what, f"{name} is on {t.device}, the logits on {device}")
    return t.data_ptr()


_WS = {}


def _workspace_bytes(tag, rows, vocab, by_count, device):
    """Workspace for these sizes on ``device``, cached per sizes."""
    key = (tag, rows, vocab, by_count, device.index)
    n = _WS.get(key)
    if n is None:
        if len(_WS) >= 4096:
            _WS.clear()
        got = ctypes.c_int64(0)
        with torch.cuda.device(device):
            _lib.call("vqx_sample_tokens_workspace_size", tag, rows, vocab, by_count, got)
        n = _WS[key] = got.value
    return n


@torch.library.impl(quantized_ops_lib, "sample_tokens", "CUDA")
def sample_tokens(logits, random, temperature=None, top_k=None, top_p=None, min_p=None):
    """A token for each row of logits [rows, vocab] (fp32, bf16 or fp16) from
    random (fp32 [rows], in [0, 1)).  temperature (fp32 [rows]; 0: the largest
    logit), then top_k (int32 [rows]; 0: all), top_p (fp32 [rows]; 1: all) of
    what that leaves, then min_p (fp32 [rows]; of the largest probability); None:
    1 and no cut.  Equal logits go by the lower index.  Weights are whole numbers
    of 41 bits and their sums exact, so that a row and its number give one token
    however the work is shared out.  Returns (tokens int64 [rows]: the first, by
    index, of those kept whose sum passes random's share of the total; the
    logarithm of its probability among those kept, fp32 [rows]); -1 and -inf for
    a row without a logit above -inf.  A NaN is never drawn."""
    what = "sample_tokens"
    _lib.require_device(logits, what)
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= 2 ** 22:
        kv4._refuse(what, f"logits must be [rows, 1 to 2^22], not {list(logits.shape)}")
    tag = kv4._FLOATS.get(logits.dtype)
    if tag is None:
        kv4._refuse(what, f"logits must be float32, bfloat16 or float16, not {logits.dtype}")
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    rows, vocab = logits.shape
    device = logits.device
    if random is None:
        kv4._refuse(what, "random is one number for each row")
    given = (_of_rows(random, rows, torch.float32, "random", what, device),
             _of_rows(temperature, rows, torch.float32, "temperature", what, device),
             _of_rows(top_k, rows, torch.int32, "top_k", what, device),
             _of_rows(top_p, rows, torch.float32, "top_p", what, device),
             _of_rows(min_p, rows, torch.float32, "min_p", what, device))
    tokens = random.new_empty(rows, dtype=torch.int64)
    chances = random.new_empty(rows)
    need = _workspace_bytes(tag, rows, vocab, top_k is not None, device)
    ws = random.new_empty(need, dtype=torch.uint8) if need else None  # held until the kernels that use it are enqueued
    kv4._launch("vqx_sample_tokens", logits, logits.data_ptr(), tag, rows, vocab, logits.stride(0), *given,
                tokens.data_ptr(), chances.data_ptr(), _lib.ptr(ws), need)
    return tokens, chances


@torch.library.register_fake("quantized_ops::sample_tokens")
def _(logits, random, temperature=None, top_k=None, top_p=None, min_p=None):
    return random.new_empty(logits.shape[0], dtype=torch.int64), random.new_empty(logits.shape[0])
