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

Around that step: ``kv4_reserve`` makes ``table``, ``cu``, positions and slots from
how many tokens each sequence gets; ``kv4_append_rotary`` turns queries and keys
on the way in.  With drafted tokens, ``kv4_tree_attention`` in the place of
``kv4_attention``, ``sample_tokens`` (``sampling.py``) after it, and ``kv4_accept``,
which keeps the drafted tokens that were drawn and cuts the lengths by the others.

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
    "kv4_append_rotary": (
        "kv4_append_rotary(Tensor query, Tensor key, Tensor value, Tensor(a!) codes, Tensor(b!) scales, Tensor lengths, "
        "Tensor freqs, Tensor? cu=None, Tensor? table=None, Tensor? positions=None, *, bool interleaved=False, "
        "float factor=1.0) -> Tensor"),
    "kv4_reserve": (
        "kv4_reserve(Tensor grow, Tensor(a!) lengths, Tensor(b!) table, Tensor(c!) free, Tensor(d!) count, "
        "SymInt page_size, SymInt n) -> (Tensor, Tensor, Tensor)"),
    "kv4_tree_attention": (
        "kv4_tree_attention(Tensor query, Tensor codes, Tensor scales, Tensor lengths, Tensor tree, Tensor? cu=None, "
        "int? most=None, Tensor? table=None, *, float? scale=None, float softcap=0.0, int window=0, "
        "Tensor? slopes=None) -> (Tensor, Tensor)"),
    "kv4_accept": (
        "kv4_accept(Tensor tree, Tensor drafts, Tensor sampled, Tensor(a!) codes, Tensor(b!) scales, "
        "Tensor(c!) lengths, Tensor? cu=None, Tensor? table=None) -> (Tensor, Tensor, Tensor)"),
}
for _s in _SCHEMAS.values():
    quantized_ops_lib.define(_s)


def _impl(name):
    return torch.library.impl(quantized_ops_lib, name, "CUDA")


_FLOATS = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


_FP32_MAX, _FP32_TINY = torch.finfo(torch.float32).max, torch.finfo(torch.float32).tiny


def _refuse(what, message):
    raise ValueError(f"vqx: {what}: {message}")


def _launch(name, t, *args):
    """The library's entry point on t's device and that device's current stream."""
    stream, at = _lib.stream_of(t), t.device.index
    if at is None or at == torch.cuda.current_device():
        _lib.call(name, *args, stream)
    else:
        with torch.cuda.device(at):
            _lib.call(name, *args, stream)


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


def _turn(freqs, positions, n, dim, interleaved, factor, back, what, device):
    """How pairs are turned, as the library takes it; positions: None for places
    in a cache."""
    if freqs.dtype != torch.float32 or freqs.dim() != 1 or not freqs.is_contiguous():
        _refuse(what, f"freqs must be a contiguous float32 vector, not {freqs.dtype} {list(freqs.shape)}")
    pairs = freqs.shape[0]
    if not 1 <= pairs <= dim // 2:
        _refuse(what, f"{pairs} frequencies for the pairs of a head of {dim}")
    if freqs.device != device:
        _refuse(what, f"freqs are on {freqs.device}, the heads on {device}")
    if not -_FP32_MAX <= factor <= _FP32_MAX:
        _refuse(what, f"a factor is finite in float32, not {factor}")
    at = None if positions is None else _int32(positions, n, "positions", what, device)
    return _lib.VqxTurn(freqs.data_ptr(), at, pairs, interleaved, back, factor)


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


@_impl("kv4_append_rotary")
def kv4_append_rotary(query, key, value, codes, scales, lengths, freqs, cu=None, table=None, positions=None, *,
                      interleaved=False, factor=1.0):
    """``rotary`` of the new tokens' queries [n, heads, D], which are returned,
    and of their keys, which go into the cache with the values as by
    ``kv4_append``, in one launch.  positions: int32 [n], or None for the tokens'
    places in the cache; in one that ``kv4_evict`` has thinned out a place is no
    position."""
    what = "kv4_append_rotary"
    _lib.require_device(codes, what)
    c = _cache(codes, scales, lengths, table, what)
    device, kv, dim = codes.device, c.kv_heads, c.dim
    q, qn, qh, qtag = _rows(query, None, dim, "query", what, device)
    k, kn, kh, tag = _rows(key, kv, dim, "key", what, device)
    v, vn, vh, vtag = _rows(value, kv, dim, "value", what, device)
    n, heads, _ = q.shape
    if k.shape[0] != n or v.shape[0] != n or qtag != tag or vtag != tag:
        _refuse(what, f"query, key and value differ: {query.dtype} {list(query.shape)}, {key.dtype} {list(key.shape)}, "
                      f"{value.dtype} {list(value.shape)}")
    if heads == 0:
        _refuse(what, "0 query heads")
    offsets = _offsets(cu, n, c.seqs, what, device)
    t = _turn(freqs, positions, n, dim, interleaved, factor, False, what, device)
    out = q.new_empty((n, heads, dim))
    _launch("vqx_kv4_append_rotary", codes, c, t, q.data_ptr(), heads, qn, qh, k.data_ptr(), kn, kh, v.data_ptr(), vn,
            vh, tag, n, offsets, out.data_ptr())
    return out


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


def _workspace_bytes(c, qs, device, key, entry="vqx_kv4_attention"):
    """Workspace that entry point needs for these sizes on ``device`` (0: no
    splits to join), cached per sizes."""
    key = (c.pages_per_seq, c.page_size, c.kv_heads, c.dim, c.seqs, device.index, entry, key)
    n = _WS.get(key)
    if n is None:
        if len(_WS) >= 4096:
            _WS.clear()
        got = ctypes.c_int64(0)
        with torch.cuda.device(device):
            _lib.call(entry + "_workspace_size", c, qs, got)
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


@_impl("kv4_tree_attention")
def kv4_tree_attention(query, codes, scales, lengths, tree, cu=None, most=None, table=None, *, scale=None, softcap=0.0,
                       window=0, slopes=None):
    """kv4_attention of new tokens that are a tree of drafts, 64 of a sequence at
    most (``most``, where there are more in all).  tree (int64 [n]): bit j of a
    token's mask says that it sees its sequence's new token j: its ancestors and
    itself.  All see the cached tokens before the new ones.  For ``window`` and
    ``slopes`` a token stands as far behind those as it has ancestors, and an
    ancestor as far before it as there are others between.  Bits of tokens that
    the sequence does not have, or beyond ``most``, do not count."""
    what = "kv4_tree_attention"
    _lib.require_device(codes, what)
    c = _cache(codes, scales, lengths, table, what)
    device = codes.device
    qs, q, key = _query(query, c, device, cu, most, scale, softcap, window, slopes, what)
    n = key[0]
    masks = _int64(tree, n, "tree", what, device)
    longest = n // c.seqs if cu is None and c.seqs else qs.most or n
    if longest > 64:
        _refuse(what, f"up to {longest} new tokens of a sequence, 64 at most (say most if none has more)")
    out = q.new_empty(q.shape)
    lse = q.new_empty(key[:2], dtype=torch.float32)
    need = _workspace_bytes(c, qs, device, key, "vqx_kv4_tree_attention")
    ws = codes.new_empty(need) if need else None  # held until the kernels that use it are enqueued
    _launch("vqx_kv4_tree_attention", codes, c, qs, masks, out.data_ptr(), lse.data_ptr(), _lib.ptr(ws), need)
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


@_impl("kv4_reserve")
def kv4_reserve(grow, lengths, table, free, count, page_size, n):
    """Pages for the new tokens of a step.  grow (int32 [sequences]): how many
    tokens each sequence gets, below 0 where it ends; free (int32 [pages]): page
    numbers, the first count (int32 [1]) of them free; table: -1 where a sequence
    has no page.  Sequences that end give their pages back (behind the free ones,
    in their order; row -1, length 0).  Then each is given, from the end of the
    free ones, the pages that its new tokens lack, and its length grows.  One
    without the room in its row is passed over; from the first on that the free
    pages do not last for, or whose tokens do not fit into n, none gets a page (or
    tokens past n).  Returns (cu int32 [sequences + 1]: offsets of the new tokens
    of those that were served, positions int32 [n]: their places in their
    sequences, slots int64 [n]: page * page_size + place in the page); positions
    and slots are -1 past the last new token.  Slots are for what a program keeps of
    each token beside the cache, under the same table; the operators here take the
    table itself."""
    what = "kv4_reserve"
    _lib.require_device(lengths, what)
    device = lengths.device
    if lengths.dim() != 1:
        _refuse(what, f"lengths must be [sequences], not {list(lengths.shape)}")
    seqs = lengths.shape[0]
    if table.dim() != 2 or table.shape[0] != seqs or table.dtype != torch.int32 or not table.is_contiguous():
        _refuse(what, f"table must be a contiguous int32 tensor [{seqs}, pages of a sequence], not {table.dtype} "
                      f"{list(table.shape)}")
    if table.device != device:
        _refuse(what, f"table is on {table.device}, the lengths on {device}")
    if free.dim() != 1:
        _refuse(what, f"free must be [pages], not {list(free.shape)}")
    if n < 0:
        _refuse(what, f"{n} new tokens")
    given = (_int32(grow, seqs, "grow", what, device), _int32(lengths, seqs, "lengths", what, device), table.data_ptr(),
             _int32(free, free.shape[0], "free", what, device), _int32(count, 1, "count", what, device))
    cu, positions = lengths.new_empty(seqs + 1), lengths.new_empty(n)
    slots = lengths.new_empty(n, dtype=torch.int64)
    _launch("vqx_kv4_reserve", lengths, *given, seqs, table.shape[1], free.shape[0], page_size, n, cu.data_ptr(),
            positions.data_ptr(), slots.data_ptr())
    return cu, positions, slots


def _int64(t, n, name, what, device):
    """The address of t, a contiguous int64 vector of n on the cache's device."""
    if t.dtype != torch.int64 or t.shape != (n,) or not t.is_contiguous():
        _refuse(what, f"{name} must be a contiguous int64 tensor of shape [{n}], not {t.dtype} {list(t.shape)}")
    if t.device != device:
        _refuse(what, f"{name} is on {t.device}, the cache on {device}")
    return t.data_ptr()


@_impl("kv4_accept")
def kv4_accept(tree, drafts, sampled, codes, scales, lengths, cu=None, table=None):
    """Keep the drafted tokens that the model confirms.  tree (int64 [n]): as
    kv4_tree_attention takes it; drafts (int64 [n]): the new tokens' numbers;
    sampled (int64 [n]): what comes after each.  A sequence's first new token is
    accepted; then, from the accepted token i on, the first j > i with tree[j] ==
    tree[i] | 1 << j (a child of i) and drafts[j] == sampled[i], until there is
    none.  Their keys and values are moved to the front of the sequence's new
    tokens, and lengths is cut by the others.  Returns (path int32 [n]: at the i-th
    new token of a sequence which of them was accepted as the i-th, -1 past the
    last; how many were, int32 [sequences]; the token that comes next, int64
    [sequences], -1 where there were no new ones)."""
    what = "kv4_accept"
    _lib.require_device(codes, what)
    c = _cache(codes, scales, lengths, table, what)
    device = codes.device
    if tree.dim() != 1:
        _refuse(what, f"tree must be [new tokens], not {list(tree.shape)}")
    n = tree.shape[0]
    offsets = _offsets(cu, n, c.seqs, what, device)
    given = [_int64(t, n, name, what, device) for t, name in ((tree, "tree"), (drafts, "drafts"), (sampled, "sampled"))]
    path, accepted = lengths.new_empty(n), lengths.new_empty(c.seqs)
    follows = sampled.new_empty(c.seqs)
    _launch("vqx_kv4_accept", codes, c, *given, n, offsets, path.data_ptr(), accepted.data_ptr(), follows.data_ptr())
    return path, accepted, follows


# ---------------------------------------------------------------------------
# fake (meta) implementations for tracing
# ---------------------------------------------------------------------------
@torch.library.register_fake("quantized_ops::kv4_append")
def _(key, value, codes, scales, lengths, cu=None, table=None):
    return None


@torch.library.register_fake("quantized_ops::kv4_append_rotary")
def _(query, key, value, codes, scales, lengths, freqs, cu=None, table=None, positions=None, **kwargs):
    return query.new_empty(query.shape)


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


@torch.library.register_fake("quantized_ops::kv4_reserve")
def _(grow, lengths, table, free, count, page_size, n):
    return lengths.new_empty(lengths.shape[0] + 1), lengths.new_empty(n), lengths.new_empty(n, dtype=torch.int64)


@torch.library.register_fake("quantized_ops::kv4_accept")
def _(tree, drafts, sampled, codes, scales, lengths, cu=None, table=None):
    return lengths.new_empty(tree.shape[0]), torch.empty_like(lengths), sampled.new_empty(lengths.shape[0])


@torch.library.register_fake("quantized_ops::kv4_tree_attention")
def _(query, codes, scales, lengths, tree, cu=None, most=None, table=None, **kwargs):
    return query.new_empty(query.shape), query.new_empty(query.shape[:2], dtype=torch.float32)
