"""The operators of a serving cache held in 4 bits, and their plain forms.

The cache holds keys and values in the fp4_e2m1 microscaling format: blocks of
32 along the head dimension, one E8M0 scale byte each.  ``codes`` is uint8
[2, pages, kv heads, page size, D / 2] (keys, then values; element 2i in the
low nibble) and ``scales`` uint8 [2, pages, kv heads, page size, D / 32].  With
a block table (int32 [sequences, pages per sequence]) token t of sequence b
lives at slot t % page size of page table[b, t // page size]; without one, page
b is sequence b.  ``lengths`` counts the tokens of each sequence, those of the
current call included, so the last query of sequence b stands at lengths[b] - 1.

Kinds of case (``case["kind"]``):

* ``append``   new keys and values quantized into the cache, then read back;
* ``decode``   attention of one new token for each sequence over its cache;
* ``prompt``   attention of many new tokens for each sequence over its cache,
               each token seeing what is before it;
* ``weigh``    attention, and its weights added up for each cached token;
* ``evict``    the heaviest and the latest tokens kept, in another cache, and
               the next token's attention over that one.
"""

import math

import torch

own = False

DEV = "cuda"
BLOCK = 32
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

_OPS = None


def _ops():
    """The framework's operators."""
    global _OPS
    if _OPS is None:
        import __graft_entry__

        __graft_entry__.load_package()
        _OPS = torch.ops.quantized_ops
    return _OPS


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _case(name, kind, type="bf16", seqs=1, heads=32, kv=8, dim=128, new=1, ragged=False, length=1024, spread=0.0,
          page=0, softcap=0.0, window=0, bias=False, budget=0, recent=0):
    """new: new tokens of each sequence (the most of any, if ragged); length:
    the longest sequence, new tokens included; spread: sequences are between
    (1 - spread) * length and length long; page 0: no block table."""
    c = dict(kind=kind, type=type, seqs=seqs, heads=heads, kv=kv, dim=dim, new=new, ragged=ragged, length=length,
             spread=spread, page=page, softcap=softcap, window=window, bias=bias, budget=budget, recent=recent)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # the cache writes of one decode step of a small batch
        _case("append 16x1", "append", seqs=16, length=2048, spread=0.5, page=64),
        # ragged prompts of an admission, the projection's output cut into keys and values
        _case("append 8x2049", "append", seqs=8, kv=32, new=2049, ragged=True, length=2500, spread=0.3, page=128),
        # one sequence that has just begun, every head with keys of its own
        _case("decode 1x77 f32", "decode", type="f32", seqs=1, heads=12, kv=12, dim=64, length=77),
        # an ordinary batch of a server, grouped heads, pages
        _case("decode 16x4000", "decode", seqs=16, length=4000, spread=0.9, page=64),
        # one long document, few rows for many tokens
        _case("decode 1x131073 f16", "decode", type="f16", seqs=1, length=131073),
        # a full batch, every head with keys of its own
        _case("decode 64x4096", "decode", seqs=64, heads=32, kv=32, length=4096, spread=0.25),
        # a chunk of a prompt on top of what is cached, scores capped, window
        _case("prompt 4x300", "prompt", seqs=4, heads=16, kv=4, dim=64, new=300, ragged=True, length=5000, spread=0.6,
              page=32, softcap=30.0, window=1024),
        # a long prompt in one call
        _case("prompt 1x8192", "prompt", seqs=1, new=8192, length=8192),
        # one decode step that keeps count of what is attended to
        _case("weigh 8x2000", "weigh", seqs=8, length=2000, spread=0.5, page=64),
        # the last tokens of a prompt say which of it to keep
        _case("weigh 2x65x16385", "weigh", seqs=2, new=65, length=16385, spread=0.1),
        # a small cache that has grown over its budget
        _case("evict 8x640", "evict", seqs=8, length=640, spread=0.2, page=64, budget=512, recent=64),
        # prompts cut down to the budget of their decode cache
        _case("evict 4x50001", "evict", seqs=4, length=50001, spread=0.3, page=128, budget=8192, recent=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "weigh", "evict"])
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 2, 4, 5, 8])
    type_ = rng.choice(["bf16", "bf16", "f16", "f32"])
    page = rng.choice([0, 16, 64, 256])
    spread = rng.choice([0.0, 0.3, 0.9])
    seqs = _log(rng, 1, 48)
    room = 40_000_000 // (seqs * kv * dim)  # tokens a sequence
    args = dict(type=type_, heads=kv * group, kv=kv, dim=dim, page=page, spread=spread)
    if kind == "append":
        new = rng.choice([1, _log(rng, 2, max(2, min(4000, room // 4)))])
        return _case(None, kind, seqs=seqs, new=new, ragged=new > 1 and rng.random() < 0.5,
                     length=new + _log(rng, 1, 2000), **args)
    if kind == "prompt":
        seqs = min(seqs, 8)
        new = _log(rng, 2, max(2, min(3000, 12000 // seqs)))
        return _case(None, kind, seqs=seqs, new=new, ragged=rng.random() < 0.5, length=new + _log(rng, 1, 4000),
                     softcap=rng.choice([0.0, 0.0, 50.0]), window=rng.choice([0, 0, 700]), bias=rng.random() < 0.3,
                     **args)
    length = _log(rng, 16, max(16, min(100_000, room)))
    if kind == "evict":
        budget = max(8, int(length * rng.uniform(0.1, 0.9)))
        return _case(None, kind, seqs=seqs, length=length, budget=budget, recent=int(budget * rng.uniform(0.0, 0.5)),
                     **args)
    new = 1 if kind == "decode" else rng.choice([1, 1, _log(rng, 2, min(16, length))])
    return _case(None, kind, seqs=seqs, new=new, length=length, softcap=rng.choice([0.0, 0.0, 50.0]),
                 window=rng.choice([0, 0, 700]), bias=rng.random() < 0.3, **args)


# ---------------------------------------------------------------------------
# what a user's program has in hand
# ---------------------------------------------------------------------------
def _sizes(case):
    """(lengths, new tokens) of the sequences, on the host: the case's own, for
    every seed, so that outputs have one shape."""
    n, new, length = case["seqs"], case["new"], case["length"]
    u = torch.rand(2, n, generator=torch.Generator().manual_seed(length))
    u[0, 0] = 0.0  # the longest
    lens = (length * (1 - case["spread"] * u[0])).round().long().clamp(min=1)
    t = (new * (0.05 + 0.95 * u[1])).round().long().clamp(min=1) if case["ragged"] else torch.full((n,), new)
    if case["ragged"]:
        t[0] = new
    return torch.maximum(lens, t), t


def _channel_scale(shape, gen):
    """Channels of keys and values differ in size, a few by much."""
    s = torch.exp(0.3 * torch.randn(shape, device=DEV, generator=gen))
    return torch.where(torch.rand(shape, device=DEV, generator=gen) < 0.03, 4 * s, s)


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(DEV).manual_seed(seed)
    dt, kv, dim, seqs = TYPES[case["type"]], case["kv"], case["dim"], case["seqs"]
    lens, new = _sizes(case)
    s = dict(case=case, scale=dim ** -0.5)
    s["lengths"] = lens.to(device=DEV, dtype=torch.int32)
    cu = torch.zeros(seqs + 1, dtype=torch.int64)
    cu[1:] = new.cumsum(0)
    total = int(cu[-1])
    s["cu"] = cu.to(device=DEV, dtype=torch.int32) if case["ragged"] else None
    capacity = case["length"]

    def table(tokens):
        if not case["page"]:
            return None, seqs, tokens
        each = -(-tokens // case["page"])
        ids = torch.randperm(seqs * each + 3, generator=host)[: seqs * each].reshape(seqs, each)
        return ids.to(device=DEV, dtype=torch.int32), seqs * each + 3, case["page"]

    def empty(pages, size):
        return (torch.zeros(2, pages, kv, size, dim // 2, dtype=torch.uint8, device=DEV),
                torch.zeros(2, pages, kv, size, dim // BLOCK, dtype=torch.uint8, device=DEV))

    s["table"], pages, size = table(capacity)
    s["codes"], s["scales"] = empty(pages, size)
    channel = _channel_scale((2, kv, 1, dim), gen)
    if case["kind"] != "append":
        for p in range(0, pages, max(1, 40_000_000 // (kv * size * dim))):
            q = min(pages, p + max(1, 40_000_000 // (kv * size * dim)))
            x = torch.randn(2, q - p, kv, size, dim, device=DEV, generator=gen) * channel[:, None]
            s["codes"][:, p:q], s["scales"][:, p:q] = _quantize(x.to(torch.bfloat16))
    # one projection's output, cut into queries, keys and values
    heads = case["heads"]
    qkv = torch.randn(total, heads + 2 * kv, dim, device=DEV, generator=gen)
    qkv[:, heads:heads + kv] *= channel[0, :, 0]
    qkv[:, heads + kv:] *= channel[1, :, 0]
    qkv[:, :heads] *= 1.5
    s["qkv"] = qkv.to(dt)
    s["slopes"] = (torch.exp2(-8.0 * torch.arange(1, heads + 1, device=DEV) / heads).float() if case["bias"] else None)
    if case["kind"] == "weigh":
        s["weights"] = torch.rand(seqs, kv, capacity, device=DEV, generator=gen)
    if case["kind"] == "evict":
        # a few tokens have most of the weight; many have been seen by none
        w = torch.exp(3 * torch.randn(seqs, kv, capacity, device=DEV, generator=gen)) * 1e-2
        s["weights"] = torch.where(torch.rand(w.shape, device=DEV, generator=gen) < 0.1, 0.0, w)
        s["out_table"], pages, size = table(case["budget"])
        s["out_codes"], s["out_scales"] = empty(pages, size)
        s["out_weights"] = torch.zeros(seqs, kv, case["budget"], device=DEV)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _quantize(x):
    """Codes and scale bytes of x along its last axis: the scale is
    2 ** (floor(log2(largest magnitude)) - 2), the log in x's own type (fp16
    in fp32), and values go to the nearest level, ties to the even code."""
    t = torch.float32 if x.dtype == torch.float16 else x.dtype
    b = x.float().reshape(*x.shape[:-1], -1, BLOCK)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.log2(torch.where(amax == 0, 2.0 ** -126, amax)).to(t).float().floor() - 2
    e = e.clamp(-127, 127)
    v = (b * torch.exp2(-e)).to(torch.bfloat16).float()
    a = v.abs()
    # the borders between levels; one that lies on a border goes to the even code
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = (code | (torch.signbit(v).int() << 3)).to(torch.uint8).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).squeeze(-1).to(torch.uint8)


def _levels(dtype):
    v = torch.tensor(LEVELS + [-x for x in LEVELS], dtype=dtype, device=DEV)
    i = torch.arange(256, device=DEV)
    return torch.stack([v[i & 15], v[i >> 4]], -1)


def _values(codes, scales, dtype=torch.float32):
    """What codes [..., D / 2] and scales [..., D / 32] stand for."""
    v = _levels(dtype)[codes.int()].reshape(*scales.shape, BLOCK)
    return (v * torch.exp2(scales.to(dtype) - 127)[..., None]).flatten(-2)


def _place(table, size, b, t):
    """(page, slot) of token t of sequence b."""
    return (b.expand_as(t), t) if table is None else (table.long()[b, t // size], t % size)


def _new_tokens(s):
    """(sequence, position) of each new token."""
    c, n = s["case"], s["qkv"].shape[0]
    i = torch.arange(n, device=DEV)
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(c["seqs"] + 1, device=DEV) * c["new"]
    b = torch.searchsorted(cu, i, right=True) - 1
    return b, s["lengths"].long()[b] - (cu[b + 1] - i)


def _gathered(plane, table, n, tokens):
    """[n, kv, tokens, x] of one plane [pages, kv, size, x]."""
    if table is None:
        return plane[:, :, :tokens]
    kv, size, x = plane.shape[1:]
    return plane[table.long()].transpose(1, 2).reshape(n, kv, -1, x)[:, :, :tokens]


def _parts(s):
    h, kv = s["case"]["heads"], s["case"]["kv"]
    return s["qkv"][:, :h], s["qkv"][:, h:h + kv], s["qkv"][:, h + kv:]


def _scores(s, q, k, lengths, slopes=True):
    """Masked scores [B, kv, T, group, tokens] of queries q [N, heads, D] on
    keys k [B, kv, tokens, D], and the place of each query in [B, T]."""
    c = s["case"]
    kv, group, tokens = c["kv"], c["heads"] // c["kv"], k.shape[2]
    b, pos = _new_tokens(dict(s, lengths=lengths))
    t = pos - lengths.long()[b] + c["new"]  # aligned to the end
    qp = torch.zeros(c["seqs"], c["new"], c["heads"], c["dim"], device=DEV)
    qp[b, t] = q.float()
    at = torch.full((c["seqs"], c["new"]), -1, device=DEV)
    at[b, t] = pos
    qp = qp.reshape(c["seqs"], c["new"], kv, group, c["dim"]).transpose(1, 2)
    x = torch.matmul(qp.reshape(c["seqs"], kv, -1, c["dim"]), k.transpose(-1, -2)) * s["scale"]
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    x = x.reshape(c["seqs"], kv, c["new"], group, tokens)
    j = torch.arange(tokens, device=DEV)
    away = (at[:, :, None] - j)[:, None, :, None]
    if s["slopes"] is not None:
        x = x - s["slopes"].reshape(1, kv, 1, group, 1) * away
    seen = (away >= 0) & (away < c["window"]) if c["window"] else away >= 0
    return x.masked_fill_(~seen, -math.inf), (b, t)


def _attend(s, q, codes, scales, table, lengths, tokens):
    """(out, lse, weights [B, kv, T, group, tokens]) of the plain attention."""
    c = s["case"]
    k, v = (_values(_gathered(codes[i], table, c["seqs"], tokens), _gathered(scales[i], table, c["seqs"], tokens))
            for i in (0, 1))
    x, (b, t) = _scores(s, q, k, lengths)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    del x
    z = p.sum(-1, keepdim=True)
    lse = (m + torch.log(z)).squeeze(-1)
    p /= torch.where(z == 0, 1.0, z)
    o = torch.matmul(p.reshape(c["seqs"], c["kv"], -1, tokens), v).reshape(*p.shape[:-1], c["dim"])
    back = lambda y: y.transpose(1, 2).flatten(2, 3)[b, t]  # noqa: E731
    return back(o).to(q.dtype), back(lse), p


def _kept(w, lengths, budget, recent):
    """(index [B, kv, budget] with -1 past the end, new lengths)."""
    n = lengths.long()[:, None, None]
    j = torch.arange(w.shape[-1], device=DEV)
    key = torch.where(j >= n - recent, math.inf, w)
    key = torch.where(j >= n, -math.inf, key)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    index = torch.sort(torch.where(order < n, order, w.shape[-1]), dim=-1).values
    return torch.where(index < n, index, -1).int(), lengths.clamp(max=budget)


def run(s):
    c = s["case"]
    q, key, value = _parts(s)
    codes, scales, lengths, cu, table = s["codes"], s["scales"], s["lengths"], s["cu"], s["table"]
    if own:
        o = _ops()
        if c["kind"] == "append":
            o.kv4_append(key, value, codes, scales, lengths, cu, table)
            return o.kv4_read(codes, scales, lengths, key.shape[0], cu, table, key.dtype)
        most = c["new"] if cu is not None else None
        how = dict(scale=s["scale"], softcap=c["softcap"], window=c["window"], slopes=s["slopes"])
        if c["kind"] == "evict":
            index, kept = o.kv4_evict(codes, scales, s["weights"], lengths, c["budget"], c["recent"], s["out_codes"],
                                      s["out_scales"], s["out_weights"], table, s["out_table"])
            out, lse = o.kv4_attention(q, s["out_codes"], s["out_scales"], kept, cu, most, s["out_table"], **how)
            return index, kept, s["out_weights"], out, lse
        out, lse = o.kv4_attention(q, codes, scales, lengths, cu, most, table, **how)
        if c["kind"] != "weigh":
            return out, lse
        w = s["weights"].clone()
        o.kv4_accumulate(q, lse, codes, scales, lengths, w, cu, most, table, **how)
        return out, lse, w
    size, tokens = codes.shape[3], c["length"]
    if c["kind"] == "append":
        page, slot = _place(table, size, *_new_tokens(s))
        read = []
        for i, x in enumerate((key, value)):
            codes[i][page, :, slot], scales[i][page, :, slot] = _quantize(x)
            read.append(_values(codes[i][page, :, slot], scales[i][page, :, slot]).to(x.dtype))
        return tuple(read)
    if c["kind"] == "evict":
        index, kept = _kept(s["weights"], lengths, c["budget"], c["recent"])
        live = index >= 0
        i = index.long().clamp(min=0)
        b = torch.arange(c["seqs"], device=DEV)[:, None, None]
        h = torch.arange(c["kv"], device=DEV)[None, :, None]
        page, slot = _place(table, size, b, i)
        j = torch.arange(c["budget"], device=DEV).expand_as(i)
        to, at = _place(s["out_table"], s["out_codes"].shape[3], b, j)
        h = h.expand_as(i)
        for x in (0, 1):
            s["out_codes"][x][to[live], h[live], at[live]] = codes[x][page[live], h[live], slot[live]]
            s["out_scales"][x][to[live], h[live], at[live]] = scales[x][page[live], h[live], slot[live]]
        s["out_weights"].copy_(torch.where(live, s["weights"].gather(-1, i), 0.0))
        out, lse, _ = _attend(s, q, s["out_codes"], s["out_scales"], s["out_table"], kept, c["budget"])
        return index, kept, s["out_weights"], out, lse
    out, lse, p = _attend(s, q, codes, scales, table, lengths, tokens)
    if c["kind"] != "weigh":
        return out, lse
    return out, lse, s["weights"] + p.sum((2, 3))


# ---------------------------------------------------------------------------
# in 64 bits, one sequence and head at a time
# ---------------------------------------------------------------------------
def _exact_values(codes, scales):
    """[tokens, D] in 64 bits from codes [tokens, D / 2] and scales: a code is
    sign, two exponent bits and one of the fraction."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    sign = torch.where(c >= 8, -1.0, 1.0)
    m = c % 8
    e = torch.div(m, 2, rounding_mode="floor")
    f = m % 2
    level = torch.where(e == 0, f / 2, torch.pow(2.0, e - 1) * (1 + f / 2))
    x = torch.ldexp(torch.ones((), dtype=torch.float64, device=DEV), scales.double() - 127)
    return sign * level * x.repeat_interleave(BLOCK, -1)


def _exact_attention(s, codes, scales, table, lengths, weigh=False):
    """(out, lse, weights added) of every query."""
    c = s["case"]
    q = _parts(s)[0].double()
    out, lse = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    added = s["weights"].double().clone() if weigh else None
    group, first = c["heads"] // c["kv"], 0
    cu = s["cu"].tolist() if s["cu"] is not None else [i * c["new"] for i in range(c["seqs"] + 1)]
    for b, n in enumerate(lengths.tolist()):
        first, end = cu[b], cu[b + 1]
        t = torch.arange(n, device=DEV)
        page, slot = _place(table, codes.shape[3], torch.tensor(b, device=DEV), t)
        pos = torch.arange(n - (end - first), n, device=DEV)
        away = pos[:, None] - t
        seen = (away >= 0) & ((away < c["window"]) if c["window"] else True)
        for h in range(c["kv"]):
            k, v = (_exact_values(codes[i][page, h, slot], scales[i][page, h, slot]) for i in (0, 1))
            for x in range(h * group, (h + 1) * group):
                a = q[first:end, x] @ k.T * s["scale"]
                if c["softcap"]:
                    a = c["softcap"] * torch.tanh(a / c["softcap"])
                if s["slopes"] is not None:
                    a = a - s["slopes"][x].double() * away
                a = a.masked_fill(~seen, -math.inf)
                z = torch.logsumexp(a, -1)
                p = torch.exp(a - z[:, None])
                out[first:end, x], lse[first:end, x] = p @ v, z
                if weigh:
                    added[b, h, :n] += p.sum(0)
    return out, lse, added


def exact(case, seed):
    s = prepare(case, seed)
    q, key, value = _parts(s)
    if case["kind"] == "append":
        level = torch.tensor(LEVELS, dtype=torch.float64, device=DEV)
        found = []
        for x in (key, value):
            b = x.double().unflatten(-1, (-1, BLOCK))
            t = torch.float32 if x.dtype == torch.float16 else x.dtype
            e = torch.log2(b.abs().amax(-1, keepdim=True)).to(t).double().floor() - 2
            v = torch.ldexp(b, -e).to(torch.bfloat16).double()
            far = (v.abs()[..., None] - level).abs()
            # of two levels as near, the one with the even code
            pick = (far + 1e-12 * (torch.arange(8, device=DEV) % 2)).argmin(-1)
            found.append(torch.ldexp(torch.copysign(level[pick], v), e).flatten(-2))
        return tuple(found)
    if case["kind"] == "evict":
        w, codes, scales = s["weights"].tolist(), s["out_codes"], s["out_scales"]
        kept = s["lengths"].clamp(max=case["budget"])
        ow = torch.zeros(s["out_weights"].shape, dtype=torch.float64)
        for b, n in enumerate(s["lengths"].tolist()):
            for h in range(case["kv"]):
                old = max(0, n - case["recent"])
                room = min(n, case["budget"]) - (n - old)
                keep = sorted(sorted(range(old), key=lambda i: (-w[b][h][i], i))[:room]) + list(range(old, n))
                m = len(keep)
                i = torch.tensor(keep, device=DEV)
                page, slot = _place(s["table"], s["codes"].shape[3], torch.tensor(b, device=DEV), i)
                to, at = _place(s["out_table"], codes.shape[3], torch.tensor(b, device=DEV), torch.arange(m, device=DEV))
                for x in (0, 1):
                    codes[x][to, h, at], scales[x][to, h, at] = s["codes"][x][page, h, slot], s["scales"][x][page, h, slot]
                ow[b, h, :m] = torch.tensor([w[b][h][i] for i in keep], dtype=torch.float64)
        out, lse, _ = _exact_attention(s, codes, scales, s["out_table"], kept)
        return None, None, ow, out, lse
    out, lse, w = _exact_attention(s, s["codes"], s["scales"], s["table"], s["lengths"], case["kind"] == "weigh")
    return (out, lse, w) if case["kind"] == "weigh" else (out, lse)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    lens, new = _sizes(c)
    n, size = int(new.sum()), torch.finfo(TYPES[c["type"]]).bits // 8
    token = c["kv"] * c["dim"] * 17 // 32  # bytes of a token's keys, or values
    queries = 2 * n * c["heads"] * c["dim"] * size + 4 * n * c["heads"]
    if c["kind"] == "append":
        # values in, codes out, codes in again, values out
        return {"bytes": 2 * (2 * n * token + 2 * n * c["kv"] * c["dim"] * size), "flops": 0}

    def pairs(length, t):
        """(query, key) pairs that are seen, and keys that any query sees."""
        w = c["window"] or length
        first = length - t
        full = sum(min(w, p + 1) for p in range(first, length))
        return full, min(length, t + w - 1)

    if c["kind"] == "evict":
        kept = lens.clamp(max=c["budget"])
        seen = int(kept.sum())
        flops = 4 * c["dim"] * c["heads"] * seen
        index = 4 * c["kv"] * c["seqs"] * c["budget"]
        return {"bytes": 4 * c["kv"] * int(lens.sum()) + 3 * 2 * token * seen + 2 * index + queries, "flops": flops}
    both = [pairs(int(a), int(b)) for a, b in zip(lens, new)]
    seen, keys = sum(x[0] for x in both), sum(x[1] for x in both)
    moved, flops = 2 * token * keys + queries, 4 * c["dim"] * c["heads"] * seen
    if c["kind"] == "weigh":
        moved += 8 * c["kv"] * c["seqs"] * c["length"]
    return {"bytes": moved, "flops": flops}
