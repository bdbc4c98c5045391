"""A serving cache of keys and values in 4 bits, and the attention that reads it.

``torch.ops.quantized_ops.kv4_*``, this package's own: the reference has no cache.
They are for inference: no gradient passes through them.  The cache holds keys
and values in the layout of ``quantize_mx_packed(x, "fp4_e2m1", -1, 32)``, page
by page (but for quotients of 255 / 1024, which that rounds up as the reference
does and ``kv4_append`` to the nearer 0, and for scales below E8M0's 2^-127):

* ``codes``  uint8 [2, pages, kv heads, page size, D / 2], keys then values,
  element 2 i in the low nibble; D is 64, 128 or 256;
* ``scales`` uint8 [2, pages, kv heads, page size, D / 32], E8M0, 255 for NaN;
* ``table``  int32 [sequences, pages per sequence], or None: page b is
  sequence b.  An entry outside [0, pages) is no page: what is on it is neither
  written nor attended to;
* ``lengths`` int32 [sequences]: the tokens of each, new ones included.

New tokens come one sequence after another, those of sequence b at
``cu[b]:cu[b + 1]`` (int32), or as many for each where ``cu`` is None, and stand
at the end of their sequence.  ``most`` (with ``cu``): no sequence has more of
them; without it the launch is as large as one sequence with all of them needs.

A step of a server: ``kv4_append`` the new keys and values, ``kv4_attention``
(and, where tokens are to be weighed, ``kv4_accumulate``), and where a cache
has grown over its budget ``kv4_evict`` into another one.  All of it is
enqueued on the current stream without a look at the device's data, so a decode
step can be captured into a graph and replayed as ``lengths`` grows.  Since the
lengths are not looked at, work is shared out as if each sequence filled its
room (the table's pages): a table many times as wide as the sequences costs up
to four times the time.

A place is a slot of the cache.  ``kv4_evict`` moves the kept tokens to the
front, for each kv head others, so that in a cache that it has filled distances
are of slots: ``window`` and ``slopes`` no longer count the tokens that were
between.
"""

import ctypes
import math

import torch

from .. import _lib
from .quantized import quantized_ops_lib

_SCHEMAS = {
    "kv4_append": (
        "kv4_append(Tensor key, Tensor value, Tensor(a!) codes, Tensor(b!) scales, Tensor lengths, "
        "Tensor? cu=None, Tensor? table=None) -> ()"),
    "kv4_read": (
        "kv4_read(Tensor codes, Tensor scales, Tensor lengths, SymInt n, Tensor? cu=None, Tensor? table=None, "
        "ScalarType dtype=bfloat16) -> (Tensor, Tensor)"),
    "kv4_attention": (
        "kv4_attention(Tensor query, Tensor codes, Tensor scales, Tensor lengths, Tensor? cu=None, int? most=None, "
        "Tensor? table=None, *, float? scale=None, float softcap=0.0, int window=0, Tensor? slopes=None) "
        "-> (Tensor, Tensor)"),
    "kv4_accumulate": (
        "kv4_accumulate(Tensor query, Tensor lse, Tensor codes, Tensor scales, Tensor lengths, Tensor(a!) weights, "
        "Tensor? cu=None, int? most=None, Tensor? table=None, *, float? scale=None, float softcap=0.0, "
        "int window=0, Tensor? slopes=None) -> ()"),
    "kv4_evict": (
        "kv4_evict(Tensor codes, Tensor scales, Tensor weights, Tensor lengths, int budget, int recent, "
        "Tensor(a!) out_codes, Tensor(b!) out_scales, Tensor(c!) out_weights, Tensor? table=None, "
        "Tensor? out_table=None) -> (Tensor, Tensor)"),
}
for _s in _SCHEMAS.values():
    quantized_ops_lib.define(_s)


def _impl(name):
    return torch.library.impl(quantized_ops_lib, name, "CUDA")


_FLOATS = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


_FP32_MAX, _FP32_TINY = torch.finfo(torch.float32).max, torch.finfo(torch.float32).tiny


def _refuse(what, message):
    raise ValueError(f"vqx: {what}: {message}")


def _int32(t, n, name, what, device):
    """The address of t, a contiguous int32 vector of n on the cache's device."""
    if t.dtype != torch.int32 or t.shape != (n,) or not t.is_contiguous():
        _refuse(what, f"{name} must be a contiguous int32 tensor of shape [{n}], not {t.dtype} {list(t.shape)}")
    if t.device != device:
        _refuse(what, f"{name} is on {t.device}, the cache on {device}")
    return t.data_ptr()


def _cache(codes, scales, lengths, table, what):
    """The cache as the library takes it.  Tensors that a kernel writes or
    whose layout its indexes assume are checked, never copied."""
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        _refuse(what, f"codes and scales must be uint8, not {codes.dtype} and {scales.dtype}")
    shape = codes.shape
    if len(shape) != 5 or shape[0] != 2 or shape[4] not in (32, 64, 128):
        _refuse(what, "codes must be [2, pages, kv heads, page size, D / 2] with D 64, 128 or 256, "
                      f"not {list(shape)}")
    _, pages, kv, size, half = shape
    if scales.shape != (2, pages, kv, size, half // 16):
        _refuse(what, f"scales must be [2, pages, kv heads, page size, D / 32], not {list(scales.shape)} "
                      f"for codes {list(shape)}")
    if not (codes.is_contiguous() and scales.is_contiguous()):
        _refuse(what, "codes and scales must be contiguous")
    device = codes.device
    if scales.device != device:
        _refuse(what, f"scales are on {scales.device}, codes on {device}")
    if lengths.dim() != 1:
        _refuse(what, f"lengths must be [sequences], not {list(lengths.shape)}")
    seqs = lengths.shape[0]
    at, tab, per = _int32(lengths, seqs, "lengths", what, device), None, 0
    if table is not None:
        if table.dim() != 2 or table.shape[0] != seqs or table.dtype != torch.int32 or not table.is_contiguous():
            _refuse(what, f"table must be a contiguous int32 tensor [{seqs}, pages of a sequence], not {table.dtype} "
                          f"{list(table.shape)}")
        if table.device != device:
            _refuse(what, f"table is on {table.device}, the cache on {device}")
        per, tab = table.shape[1], table.data_ptr()
        if per == 0:
            _refuse(what, "table has no pages for a sequence")
    return _lib.VqxKv4Cache(codes.data_ptr(), scales.data_ptr(), tab, at, pages, per, kv, size, 2 * half, seqs)


def _offsets(cu, n, seqs, what, device):
    if cu is not None:
        return _int32(cu, seqs + 1, "cu", what, device)
    if n % seqs if seqs else n:
        _refuse(what, f"{n} new tokens for {seqs} sequences need cu")
    return None


def _rows(t, heads, dim, name, what, device):
    """t [n, heads, dim] with rows that start on 16 bytes, copied if they do
    not, its strides and its dtype's tag."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads):
        _refuse(what, f"{name} must be [new tokens, {'heads' if heads is None else heads}, {dim}], "
                      f"not {list(shape)}")
    tag = _FLOATS.get(t.dtype)
    if tag is None:
        _refuse(what, f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    if t.device != device:
        _refuse(what, f"{name} is on {t.device}, the cache on {device}")
    sn, sh, sd = t.stride()
    per = 3 if tag == _lib.F32 else 7  # elements of 16 bytes, less 1
    if sd != 1 or sn & per or sh & per or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        sn, sh, _ = t.stride()
    return t, sn, sh, tag


def _query(query, cache, device, cu, most, scale, softcap, window, slopes, what):
    """(the queries as the library takes them, the tensor that holds them, a
    key of all that their workspace depends on beside the cache's sizes)."""
    dim, kv, seqs = cache.dim, cache.kv_heads, cache.seqs
    q, sn, sh, tag = _rows(query, None, dim, "query", what, device)
    n, heads, _ = q.shape
    if heads == 0 or heads % kv:
        _refuse(what, f"{heads} query heads for {kv} kv heads")
    offsets = _offsets(cu, n, seqs, what, device)
    if most is None:
        most = 0
    elif most < (1 if n else 0):
        _refuse(what, f"most is {most}")
    elif most > n:
        most = n
    if not 0 <= window < 2 ** 30:
        _refuse(what, f"a window is positive and below 2^30, or 0 for none, not {window}")
    scale = dim ** -0.5 if scale is None else scale
    if not -_FP32_MAX <= scale <= _FP32_MAX:
        _refuse(what, f"a scale is finite in float32, not {scale}")
    if not 0.0 <= softcap < math.inf:
        _refuse(what, f"a softcap is positive, or 0 for none, not {softcap}")
    if softcap != 0.0 and not (_FP32_TINY <= softcap and abs(scale) <= _FP32_MAX * softcap):
        _refuse(what, f"a softcap of {softcap} is too small for a scale of {scale} in float32")
    bias = None
    if slopes is not None:
        if slopes.dtype != torch.float32 or slopes.shape != (heads,) or not slopes.is_contiguous():
            _refuse(what, f"slopes must be a contiguous float32 tensor of {heads}, not {slopes.dtype} "
                          f"{list(slopes.shape)}")
        if slopes.device != device:
            _refuse(what, f"slopes are on {slopes.device}, the cache on {device}")
        bias = slopes.data_ptr()
    return (_lib.VqxKv4Query(q.data_ptr(), offsets, bias, n, sn, sh, tag, heads, most, window,
                             scale, softcap),
            q, (n, heads, tag, most, window, cu is None))


def _weights(weights, seqs, kv, name, what, device):
    if weights.dtype != torch.float32 or weights.ndim != 3 or weights.shape[:2] != (seqs, kv) \
            or not weights.is_contiguous():
        _refuse(what, f"{name} must be a contiguous float32 tensor [{seqs}, {kv}, tokens], not {weights.dtype} "
                      f"{list(weights.shape)}")
    if weights.device != device:
        _refuse(what, f"{name} are on {weights.device}, the cache on {device}")
    return weights.data_ptr()


@_impl("kv4_append")
def kv4_append(key, value, codes, scales, lengths, cu=None, table=None):
    """Quantize the new tokens' keys and values [n, kv heads, D] into their
    places in the cache."""
    what = "kv4_append"
    _lib.require_device(codes, what)
    c = _cache(codes, scales, lengths, table, what)
    device, kv, dim = codes.device, c.kv_heads, c.dim
    k, kn, kh, tag = _rows(key, kv, dim, "key", what, device)
    v, vn, vh, vtag = _rows(value, kv, dim, "value", what, device)
    n = k.shape[0]
    if v.shape[0] != n or vtag != tag:
        _refuse(what, f"key and value differ: {key.dtype} {list(key.shape)}, {value.dtype} {list(value.shape)}")
    offsets = _offsets(cu, n, c.seqs, what, device)
    _lib.call("vqx_kv4_append", c, k.data_ptr(), v.data_ptr(), tag, n, kn, kh, vn, vh, offsets,
              _lib.stream_of(codes))


@_impl("kv4_read")
def kv4_read(codes, scales, lengths, n, cu=None, table=None, dtype=torch.bfloat16):
    """The keys and values [n, kv heads, D] of the n new tokens as the cache
    holds them."""
    what = "kv4_read"
    _lib.require_device(codes, what)
    c = _cache(codes, scales, lengths, table, what)
    if dtype not in _FLOATS:
        _refuse(what, f"float32, bfloat16 or float16 values, not {dtype}")
    if n < 0:
        _refuse(what, f"{n} new tokens")
    offsets = _offsets(cu, n, c.seqs, what, codes.device)
    k = codes.new_empty((n, c.kv_heads, c.dim), dtype=dtype)
    v = torch.empty_like(k)
    _lib.call("vqx_kv4_read", c, k.data_ptr(), v.data_ptr(), _FLOATS[dtype], n, offsets, _lib.stream_of(codes))
    return k, v


_WS = {}


def _workspace_bytes(c, qs, device, key):
    """Workspace vqx_kv4_attention needs for these sizes on ``device`` (0: no
    splits to join), cached per sizes."""
    key = (c.pages_per_seq, c.page_size, c.kv_heads, c.dim, c.seqs, device.index, key)
    n = _WS.get(key)
    if n is None:
        if len(_WS) >= 4096:
            _WS.clear()
        got = ctypes.c_int64(0)
        with torch.cuda.device(device):
            _lib.call("vqx_kv4_attention_workspace_size", c, qs, got)
        n = _WS[key] = got.value
    return n


@_impl("kv4_attention")
def kv4_attention(query, codes, scales, lengths, cu=None, most=None, table=None, *, scale=None, softcap=0.0,
                  window=0, slopes=None):
    """(out, lse) of the new tokens' queries [n, heads, D] over their
    sequences: each sees what is at or before its place, the last `window`
    tokens of it if that is not 0.  Scores are scale q.k (1 / sqrt(D)), capped to
    softcap tanh(s / softcap) if that is not 0, less slopes[head] for each
    token of distance.  out has the queries' dtype; lse [n, heads] is fp32.
    A query that sees nothing has out 0 and lse -inf."""
    what = "kv4_attention"
    _lib.require_device(codes, what)
    c = _cache(codes, scales, lengths, table, what)
    device = codes.device
    qs, q, key = _query(query, c, device, cu, most, scale, softcap, window, slopes, what)
    out = q.new_empty(q.shape)
    lse = q.new_empty(key[:2], dtype=torch.float32)
    need = _workspace_bytes(c, qs, device, key)
    ws = codes.new_empty(need) if need else None  # held until the kernels that use it are enqueued
    _lib.call("vqx_kv4_attention", c, qs, out.data_ptr(), lse.data_ptr(), _lib.ptr(ws), need, _lib.stream_of(codes))
    return out, lse


@_impl("kv4_accumulate")
def kv4_accumulate(query, lse, codes, scales, lengths, weights, cu=None, most=None, table=None, *, scale=None,
                   softcap=0.0, window=0, slopes=None):
    """Add to weights (fp32 [sequences, kv heads, tokens]) what the attention of
    these queries gives each cached token, over the new tokens and the query
    heads of a kv head; lse as kv4_attention gives it."""
    what = "kv4_accumulate"
    _lib.require_device(codes, what)
    c = _cache(codes, scales, lengths, table, what)
    qs, q, _ = _query(query, c, codes.device, cu, most, scale, softcap, window, slopes, what)
    if lse.dtype != torch.float32 or lse.shape != q.shape[:2] or not lse.is_contiguous() or lse.device != q.device:
        _refuse(what, f"lse must be a contiguous float32 tensor {list(q.shape[:2])}, not {lse.dtype} "
                      f"{list(lse.shape)}")
    w = _weights(weights, c.seqs, c.kv_heads, "weights", what, codes.device)
    _lib.call("vqx_kv4_accumulate", c, qs, lse.data_ptr(), w, weights.shape[2], _lib.stream_of(codes))


@_impl("kv4_evict")
def kv4_evict(codes, scales, weights, lengths, budget, recent, out_codes, out_scales, out_weights, table=None,
              out_table=None):
    """Keep min(budget, length) tokens of each sequence for each kv head, the
    latest `recent` and the heaviest before them, in their order at the front of
    the other cache; equal weights go by the lower place, NaN is above all.
    Returns (index int32 [sequences, kv heads, budget]: where each kept token
    was, -1 past the end; the new lengths); out_weights gets their weights (a
    heavy -0 as 0, a heavy NaN as the quiet one), 0 past the end."""
    what = "kv4_evict"
    _lib.require_device(codes, what)
    c = _cache(codes, scales, lengths, table, what)
    device = codes.device
    kept = torch.empty_like(lengths)
    o = _cache(out_codes, out_scales, kept, out_table, what)
    if out_codes.device != device:
        _refuse(what, f"the caches are on {device} and {out_codes.device}")
    if not 1 <= budget < 2 ** 31 or not 0 <= recent <= budget:
        _refuse(what, f"a budget of {budget} tokens, {recent} of them the latest")
    w = _weights(weights, c.seqs, c.kv_heads, "weights", what, device)
    ow = _weights(out_weights, c.seqs, c.kv_heads, "out_weights", what, device)
    if out_weights.shape[2] != budget:
        _refuse(what, f"out_weights are for {out_weights.shape[2]} tokens, the budget is {budget}")
    index = lengths.new_empty((c.seqs, c.kv_heads, budget))
    need = ctypes.c_int64(0)
    _lib.call("vqx_kv4_evict_workspace_size", c, weights.shape[2], need)
    need = need.value
    ws = codes.new_empty(need) if need else None  # held until the kernels that use it are enqueued
    _lib.call("vqx_kv4_evict", c, w, weights.shape[2], budget, recent, o, index.data_ptr(), ow, _lib.ptr(ws), need,
              _lib.stream_of(codes))
    return index, kept


# ---------------------------------------------------------------------------
# fake (meta) implementations for tracing
# ---------------------------------------------------------------------------
@torch.library.register_fake("quantized_ops::kv4_append")
def _(key, value, codes, scales, lengths, cu=None, table=None):
    return None


@torch.library.register_fake("quantized_ops::kv4_read")
def _(codes, scales, lengths, n, cu=None, table=None, dtype=torch.bfloat16):
    shape = (n, codes.shape[2], 2 * codes.shape[4])
    return codes.new_empty(shape, dtype=dtype), codes.new_empty(shape, dtype=dtype)


@torch.library.register_fake("quantized_ops::kv4_attention")
def _(query, codes, scales, lengths, cu=None, most=None, table=None, **kwargs):
    return query.new_empty(query.shape), query.new_empty(query.shape[:2], dtype=torch.float32)


@torch.library.register_fake("quantized_ops::kv4_accumulate")
def _(query, lse, codes, scales, lengths, weights, cu=None, most=None, table=None, **kwargs):
    return None


@torch.library.register_fake("quantized_ops::kv4_evict")
def _(codes, scales, weights, lengths, budget, recent, out_codes, out_scales, out_weights, table=None,
      out_table=None):
    return (lengths.new_empty((lengths.shape[0], codes.shape[2], budget)), torch.empty_like(lengths))
