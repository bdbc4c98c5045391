"""The operators around a 4-bit serving cache, and their plain forms.

One step of a server that decodes from the cache of ``kv4_append``: pages are
handed out, queries and keys turned to their positions, drafted tokens attended
to as a tree, tokens drawn from logits, and what was drafted rightly kept.  The
cache: ``codes`` uint8 [2, pages, kv heads, page size, D / 2] (keys, then values;
element 2i in the low nibble), ``scales`` uint8 [2, pages, kv heads, page size,
D / 32] (E8M0), ``table`` int32 [sequences, pages per sequence], ``lengths`` int32
[sequences], new tokens included and at the end; new tokens come one sequence
after another, those of sequence b at cu[b]:cu[b + 1].

Kinds of case (``case["kind"]``):

* ``place``   queries and keys turned by rotary positions, keys and values
              quantized into the cache, then read back;
* ``rotate``  the same turn alone, forward and backward, as in training;
* ``pages``   sequences end, others grow: block table, offsets, positions and
              slots of the new tokens;
* ``tree``    attention of drafted tokens, each of which sees the cached tokens
              and its own ancestors among the drafted;
* ``accept``  drafted tokens appended, the confirmed ones moved to the front of
              them, the lengths cut;
* ``sample``  a token for each row of logits from a given random number, and the
              logarithm of its probability among those that could be drawn.
"""

import math

import torch

own = False

DEV = "cuda"
BLOCK = 32
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
UNIT = 2.0 ** 40  # the weight of the likeliest token

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
def _named(name, c):
    return dict(name=name, **c) if name else c


def _place(name, kind="place", type="bf16", seqs=1, heads=32, kv=8, dim=128, turned=128, new=1, ragged=False,
           length=1024, spread=0.0, page=0, interleaved=False, stretch=1.0, moved=False):
    """turned: how much of a head is turned; stretch: the context is so many
    times the trained one; moved: positions are given, since tokens were taken
    out of the cache; spread, ragged: lengths and new tokens differ."""
    return _named(name, dict(kind=kind, type=type, seqs=seqs, heads=heads, kv=kv, dim=dim, turned=turned, new=new,
                             ragged=ragged, length=length, spread=spread, page=page, interleaved=interleaved,
                             stretch=stretch, moved=moved))


def _pages(name, seqs, per, page, spare, new, ended=0.0, prompts=0.0):
    """per: pages a sequence can have; spare: free pages for each sequence;
    prompts: the share of sequences with up to `new` tokens, the others have 1."""
    return _named(name, dict(kind="pages", seqs=seqs, per=per, page=page, spare=spare, new=new, ended=ended,
                             prompts=prompts))


def _tree(name, kind="tree", type="bf16", seqs=1, heads=32, kv=8, dim=128, new=8, ragged=False, length=1024, spread=0.0,
          page=0, softcap=0.0, window=0, bias=False):
    return _named(name, dict(kind=kind, type=type, seqs=seqs, heads=heads, kv=kv, dim=dim, new=new, ragged=ragged,
                             length=length, spread=spread, page=page, softcap=softcap, window=window, bias=bias))


def _sample(name, type, rows, vocab, temperature=True, top_k=0, top_p=False, min_p=False, pad=0):
    """top_k: the largest k of any row, 0 for no such tensor; pad: columns
    behind the vocabulary that are not part of it."""
    return _named(name, dict(kind="sample", type=type, rows=rows, vocab=vocab, temperature=temperature, top_k=top_k,
                             top_p=top_p, min_p=min_p, pad=pad))


def listed():
    return [
        # the keys and queries of one decode step of a small batch
        _place("place 16x1", seqs=16, length=4000, spread=0.9, page=64),
        # ragged prompts of an admission; half of each head turned, pairs side by side, a stretched context
        _place("place 8x2049 f16", type="f16", seqs=8, new=2049, ragged=True, length=2500, spread=0.3, page=128,
               turned=64, interleaved=True, stretch=8.0),
        # a training step's queries, forward and backward
        _place("rotate 4x2048", "rotate", seqs=4, new=2048, length=2048),
        # one decode step: a token for each sequence, a new page for a few
        _pages("pages 16x1", 16, 64, 64, 2, 1),
        # a busy server: sequences end, prompts are admitted, the others decode
        _pages("pages 512", 512, 128, 32, 40, 2000, ended=0.1, prompts=0.3),
        # a small tree on a sequence that has just begun
        _tree("tree 1x7 f32", type="f32", heads=12, kv=12, dim=64, new=7, length=90),
        # an ordinary batch, trees of some twenty tokens, grouped heads, pages
        _tree("tree 16x24", seqs=16, new=24, ragged=True, length=4000, spread=0.9, page=64),
        # wide trees on long documents, scores capped, distances weighed
        _tree("tree 8x64 f16", type="f16", seqs=8, new=64, length=33000, spread=0.2, page=128, softcap=30.0, bias=True),
        # the end of a step of a small batch
        _tree("accept 4x8", "accept", seqs=4, new=8, ragged=True, length=700, spread=0.5, page=64),
        # a full batch of wide trees, every head with keys of its own
        _tree("accept 64x64", "accept", seqs=64, heads=32, kv=32, new=64, length=600, spread=0.5, page=64),
        # one sequence, all that a user can ask for
        _sample("sample 1x32000", "f32", 1, 32000, top_k=50, top_p=True, min_p=True),
        # a full batch with a large vocabulary
        _sample("sample 256x131072", "bf16", 256, 131072, top_k=1000, top_p=True, min_p=True, pad=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["place", "rotate", "pages", "tree", "tree", "accept", "sample", "sample"])
    if kind == "sample":
        vocab = _log(rng, 2, 250_000)
        return _sample(None, rng.choice(["bf16", "f16", "f32"]), _log(rng, 1, max(1, min(512, 25_000_000 // vocab))), vocab,
                       temperature=rng.random() < 0.8, top_k=rng.choice([0, 1, 40, _log(rng, 2, 20_000)]),
                       top_p=rng.random() < 0.5, min_p=rng.random() < 0.4, pad=rng.choice([0, 0, 1, 64]))
    if kind == "pages":
        seqs, page = _log(rng, 1, 512), rng.choice([16, 32, 48, 64, 256])
        new = _log(rng, 1, 2000)
        return _pages(None, seqs, max(2, -(-2 * new // page) + rng.randrange(40)), page, rng.choice([1, 4, 60]), new,
                      ended=rng.choice([0.0, 0.2]), prompts=rng.choice([0.0, 0.2, 1.0]))
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 2, 4, 5, 8])
    args = dict(type=rng.choice(["bf16", "bf16", "f16", "f32"]), heads=kv * group, kv=kv, dim=dim,
                page=rng.choice([0, 16, 64, 100, 256]), spread=rng.choice([0.0, 0.3, 0.9]))
    if kind in ("place", "rotate"):
        new = rng.choice([1, _log(rng, 2, 2000)])
        most = max(1, min(64, 25_000_000 // (new * kv * group * dim)))
        return _place(None, kind, seqs=_log(rng, 1, most), new=new, ragged=rng.random() < 0.5,
                      length=new + _log(rng, 1, 100_000 if most > 40 and args["page"] == 0 and kv * dim < 600 else 2000),
                      turned=rng.choice([dim, dim // 2, dim // 4, 24]), interleaved=rng.random() < 0.5,
                      stretch=rng.choice([1.0, 4.0]), moved=kind == "place" and rng.random() < 0.4, **args)
    new = _log(rng, 1, 64)
    seqs = _log(rng, 1, 32)
    if kind == "accept":
        return _tree(None, kind, seqs=seqs, new=new, ragged=rng.random() < 0.5, length=new + _log(rng, 1, 800), **args)
    # scores of the plain form within some gigabytes, a cache too
    room = min(500_000_000 // (seqs * kv * group * new), 40_000_000 // (seqs * kv * dim))
    return _tree(None, kind, seqs=seqs, new=new, ragged=rng.random() < 0.5,
                 length=new + _log(rng, 1, max(16, min(60_000, room))), softcap=rng.choice([0.0, 0.0, 50.0]),
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


def _page_sizes(case):
    """(tokens so far, new tokens: -1 where a sequence ends) on the host."""
    g = torch.Generator().manual_seed(case["seqs"] + case["new"])
    n = case["seqs"]
    u = torch.rand(4, n, generator=g)
    new = torch.where(u[0] < case["prompts"], (u[1] * case["new"]).long() + 1, 1)
    new = torch.where(u[2] < case["ended"], -1, new)
    room = case["per"] * case["page"] - new.clamp(min=0)
    return (u[3] * room.clamp(min=0)).long(), new


def _frequencies(turned, stretch, base=10000.0, trained=4096):
    """How far each pair turns from one position to the next; with a stretched
    context, pairs that turn less than once within the trained one turn so many
    times slower, those that turn more than four times as before."""
    f = base ** (-torch.arange(0, turned, 2, dtype=torch.float64) / turned)
    turns = trained * f / (2 * math.pi)
    blend = ((turns - 1) / 3).clamp(0, 1)
    return (f * blend + f / stretch * (1 - blend)).float()


def _forest(new, gen):
    """int64 [tokens]: the ancestors of each drafted token, itself included, as
    bits, for sequences of `new` tokens each."""
    found = []
    for c in new.tolist():
        u = torch.rand(c, generator=gen).tolist()
        masks = [1]
        for j in range(1, c):
            parent = j - 1 if u[j] < 0.5 else int(u[j] * 2 * j) % j
            masks.append(masks[parent] | 1 << j)
        found += [m - (1 << 64) if m >> 63 else m for m in masks]
    return torch.tensor(found, dtype=torch.int64)


def _channel_scale(shape, gen):
    """Channels of keys and values differ in size, a few by much."""
    s = torch.exp(0.3 * torch.randn(shape, device=DEV, generator=gen))
    return torch.where(torch.rand(shape, device=DEV, generator=gen) < 0.03, 4 * s, s)


def _prepare_pages(case, host):
    lens, new = _page_sizes(case)
    n, per, page = case["seqs"], case["per"], case["page"]
    held = -(-lens // page)
    used = int(held.sum())
    pages = used + case["spare"] * n
    ids = torch.randperm(pages, generator=host).int()
    table = torch.full((n, per), -1, dtype=torch.int32)
    table[torch.arange(per)[None] < held[:, None]] = ids[:used]
    free = torch.zeros(pages, dtype=torch.int32)
    free[:pages - used] = ids[used:]
    s = dict(case=case, first=dict(lengths=lens.int(), table=table, free=free, count=torch.tensor([pages - used]).int()))
    s["first"] = {k: v.to(DEV) for k, v in s["first"].items()}
    s["now"] = {k: v.clone() for k, v in s["first"].items()}
    s["new"] = new.int().to(DEV)
    s["n"] = int(new.clamp(min=0).sum())
    return s


def _prepare_sample(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    x = 2.5 * torch.randn(rows, vocab + case["pad"], device=DEV, generator=gen)
    # a few tokens stand out, some are forbidden
    u = torch.rand(x.shape, device=DEV, generator=gen)
    x = torch.where(u < 30.0 / vocab, x + 6.0, x)
    x = torch.where((u > 0.97) & (u < 0.999), -math.inf, x)
    s = dict(case=case, logits=x.to(TYPES[case["type"]])[:, :vocab],
             random=torch.rand(rows, device=DEV, generator=gen))
    u = torch.rand(4, rows, device=DEV, generator=gen)
    s["temperature"] = torch.where(u[0] < 0.1, 0.0, 0.3 + 1.2 * u[0]) if case["temperature"] else None
    s["top_k"] = (1 + u[1] * case["top_k"]).int().clamp(max=case["top_k"]) if case["top_k"] else None
    s["top_p"] = torch.where(u[2] < 0.2, 1.0, 0.5 + 0.49 * u[2]) if case["top_p"] else None
    s["min_p"] = torch.where(u[3] < 0.3, 0.0, 0.1 * u[3]) if case["min_p"] else None
    return s


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(DEV).manual_seed(seed)
    if case["kind"] == "pages":
        return _prepare_pages(case, host)
    if case["kind"] == "sample":
        return _prepare_sample(case, gen)
    dt, kv, dim, seqs, heads = TYPES[case["type"]], case["kv"], case["dim"], case["seqs"], case["heads"]
    lens, new = _sizes(case)
    s = dict(case=case)
    s["lengths"] = lens.to(device=DEV, dtype=torch.int32)
    cu = torch.zeros(seqs + 1, dtype=torch.int64)
    cu[1:] = new.cumsum(0)
    total = int(cu[-1])
    s["cu"] = cu.to(device=DEV, dtype=torch.int32) if case["ragged"] else None
    if case["kind"] in ("place", "rotate"):
        s["freqs"] = _frequencies(case["turned"], case["stretch"]).to(DEV)
    if case["kind"] == "rotate":
        b, pos = _new_tokens(dict(s, tokens=total))
        s["positions"] = pos.int()
        s["x"] = torch.randn(total, heads, dim, device=DEV, generator=gen).to(dt).requires_grad_()
        s["grad"] = torch.randn(total, heads, dim, device=DEV, generator=gen).to(dt)
        return s
    # one projection's output, cut into queries, keys and values
    channel = _channel_scale((2, kv, 1, dim), gen)
    qkv = torch.randn(total, heads + 2 * kv, dim, device=DEV, generator=gen)
    qkv[:, heads:heads + kv] *= channel[0, :, 0]
    qkv[:, heads + kv:] *= channel[1, :, 0]
    qkv[:, :heads] *= 1.5
    s["qkv"] = qkv.to(dt)
    s["tokens"] = total
    size = case["page"] or case["length"]
    each = -(-case["length"] // size)
    pages = seqs * each + (3 if case["page"] else 0)
    s["table"] = (torch.randperm(pages, generator=host)[:seqs * each].reshape(seqs, each).to(device=DEV, dtype=torch.int32)
                  if case["page"] else None)
    s["codes"] = torch.zeros(2, pages, kv, size, dim // 2, dtype=torch.uint8, device=DEV)
    s["scales"] = torch.zeros(2, pages, kv, size, dim // BLOCK, dtype=torch.uint8, device=DEV)
    s["positions"] = None
    if case["kind"] == "place":
        if case["moved"]:
            b, pos = _new_tokens(s)
            gone = torch.randint(0, 100_000, (seqs,), device=DEV, generator=gen)
            s["positions"] = (pos + gone[b]).int()
        return s
    some = max(1, 40_000_000 // (kv * size * dim))
    for p in range(0, pages, some):
        q = min(pages, p + some)
        x = torch.randn(2, q - p, kv, size, dim, device=DEV, generator=gen) * channel[:, None]
        s["codes"][:, p:q], s["scales"][:, p:q] = _quantize(x.to(torch.bfloat16))
    masks = _forest(new, host)
    s["tree"] = masks.to(DEV)
    if case["kind"] == "tree":
        s["slopes"] = (torch.exp2(-8.0 * torch.arange(1, heads + 1, device=DEV) / heads).float() if case["bias"] else None)
        s["scale"] = dim ** -0.5
        return s
    # what was drafted; most of what is sampled is one of a token's children, where it has any
    drafts = torch.randint(0, 1000, (total,), generator=host)
    tokens = torch.randint(0, 1000, (total,), generator=host)
    u = torch.rand(total, generator=host).tolist()
    for b in range(seqs):
        first, c = int(cu[b]), int(new[b])
        m = [x % (1 << 64) for x in masks[first:first + c].tolist()]
        for j in range(1, c):
            parent = (m[j] ^ 1 << j).bit_length() - 1
            if u[first + j] < 0.8:
                tokens[first + parent] = drafts[first + j]
    s["drafts"], s["sampled"] = drafts.to(DEV), tokens.to(DEV)
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


def _values(codes, scales):
    """What codes [..., D / 2] and scales [..., D / 32] stand for."""
    v = torch.tensor(LEVELS + [-x for x in LEVELS], device=DEV)
    i = torch.arange(256, device=DEV)
    pairs = torch.stack([v[i & 15], v[i >> 4]], -1)
    return (pairs[codes.int()].reshape(*scales.shape, BLOCK) * torch.exp2(scales.float() - 127)[..., None]).flatten(-2)


def _slot(table, size, b, t):
    """(page, slot) of token t of sequence b."""
    return (b.expand_as(t), t) if table is None else (table.long()[b, t // size], t % size)


def _new_tokens(s):
    """(sequence, place) of each new token."""
    c = s["case"]
    i = torch.arange(s["tokens"], device=DEV)
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(c["seqs"] + 1, device=DEV) * c["new"]
    b = torch.searchsorted(cu, i, right=True) - 1
    return b, s["lengths"].long()[b] - (cu[b + 1] - i)


def _turn(x, positions, freqs, interleaved, back=False):
    """x [n, heads, D] turned to its positions, in 64 bits: the 4-bit borders
    behind it are to fall alike, and far positions have large angles."""
    r = 2 * freqs.shape[0]
    a = positions.double()[:, None] * freqs.double() * (-1 if back else 1)
    cos, sin = torch.cos(a)[:, None], torch.sin(a)[:, None]
    y = x.double()
    p, q = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., :r // 2], y[..., r // 2:r])
    u, v = p * cos - q * sin, p * sin + q * cos
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, y[..., r:]], -1).to(x.dtype)


def _parts(s):
    h, kv = s["case"]["heads"], s["case"]["kv"]
    return s["qkv"][:, :h], s["qkv"][:, h:h + kv], s["qkv"][:, h + kv:]


def _write(s, key, value):
    """The new tokens' keys and values put into the cache; their slots."""
    page, slot = _slot(s["table"], s["codes"].shape[3], *_new_tokens(s))
    for i, x in enumerate((key, value)):
        s["codes"][i][page, :, slot], s["scales"][i][page, :, slot] = _quantize(x)
    return page, slot


def _read(s, page, slot, dtype):
    return tuple(_values(s["codes"][i][page, :, slot], s["scales"][i][page, :, slot]).to(dtype) for i in (0, 1))


def _plain_pages(s):
    c, now = s["case"], s["now"]
    lengths, table, free, count, new = now["lengths"], now["table"], now["free"], now["count"], s["new"]
    page, n, pages = c["page"], s["n"], free.shape[0]
    j = torch.arange(c["per"], device=DEV)
    # the pages of sequences that end go back, in their order
    ended = (new < 0)[:, None]
    given = (ended & (table >= 0) & (table < pages)).flatten()
    at = count.long() + given.long().cumsum(0) - 1
    back = torch.cat([free, free.new_zeros(1)])
    back.scatter_(0, torch.where(given, at, pages), table.flatten())
    free.copy_(back[:pages])
    stock = count.long() + given.sum()
    table.copy_(torch.where(ended, -1, table))
    before = torch.where(ended[:, 0], 0, lengths).long()
    wanted = new.long().clamp(min=0)
    # the pages of the new tokens that a sequence lacks
    fits = before + wanted <= c["per"] * page
    first, last = before // page, -(-(before + wanted) // page)
    lack = (j >= first[:, None]) & (j < last[:, None]) & ((table < 0) | (table >= pages))
    lack &= (fits & (wanted > 0))[:, None]
    need = lack.sum(-1)
    served = fits & ((need == 0) | (need.cumsum(0) <= stock)) & (torch.where(fits, wanted, 0).cumsum(0) <= n)
    lack &= served[:, None]
    rank = lack.flatten().long().cumsum(0).reshape(lack.shape) - 1
    table.copy_(torch.where(lack, free[(stock - 1 - rank).clamp(min=0)], table))
    count.copy_(stock - lack.sum())
    added = torch.where(served, wanted, 0)
    lengths.copy_(before + added)
    cu = torch.cat([added.new_zeros(1), added.cumsum(0)])
    i = torch.arange(n, device=DEV)
    b = (torch.searchsorted(cu, i, right=True) - 1).clamp(max=c["seqs"] - 1)
    pos = before[b] + i - cu[b]
    slots = table.long()[b, (pos // page).clamp(max=c["per"] - 1)] * page + pos % page
    live = i < cu[-1]
    return cu.int(), torch.where(live, pos, -1).int(), torch.where(live, slots, -1)


def _plain_tree(s):
    """(out, lse) of the drafted tokens."""
    c = s["case"]
    q = _parts(s)[0]
    kv, group, tokens, seqs, new = c["kv"], c["heads"] // c["kv"], c["length"], c["seqs"], c["new"]
    size = s["codes"].shape[3]

    def gathered(plane):
        if s["table"] is None:
            return plane[:, :, :tokens]
        return plane[s["table"].long()].transpose(1, 2).reshape(seqs, kv, -1, plane.shape[-1])[:, :, :tokens]

    k, v = (_values(gathered(s["codes"][i]), gathered(s["scales"][i])) for i in (0, 1))
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(seqs + 1, device=DEV) * new
    b, place = _new_tokens(s)
    i = torch.arange(s["tokens"], device=DEV) - cu[b]  # which of its sequence's new tokens
    there = cu[1:] - cu[:-1]
    base = s["lengths"].long() - there
    bits = torch.zeros(seqs, new, 64, dtype=torch.bool, device=DEV)
    bit = torch.arange(64, device=DEV)
    bits[b, i] = (s["tree"][:, None] >> bit & 1).bool() & (bit < there[b, None])
    # of each row and drafted token, how many of the row's ancestors come behind it
    behind = bits.flip(-1).long().cumsum(-1).flip(-1) - bits.long()
    depth = bits.sum(-1)
    t = torch.arange(tokens, device=DEV)
    which = t - base[:, None]  # the drafted token at a place
    drafted = (which >= 0) & (which < there[:, None])
    which = which.clamp(0, 63)[:, None].expand(seqs, new, tokens)
    away = torch.where(drafted[:, None], behind.gather(-1, which), (base[:, None] + depth - 1)[..., None] - t)
    seen = torch.where(drafted[:, None], bits.gather(-1, which), t < base[:, None, None])
    if c["window"]:
        seen &= away < c["window"]
    qp = torch.zeros(seqs, new, c["heads"], c["dim"], device=DEV)
    qp[b, i] = q.float()
    qp = qp.reshape(seqs, new, kv, group, c["dim"]).transpose(1, 2).reshape(seqs, kv, -1, c["dim"])
    x = torch.matmul(qp, k.transpose(-1, -2)) * s["scale"]
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    x = x.reshape(seqs, kv, new, group, tokens)
    if s["slopes"] is not None:
        x = x - s["slopes"].reshape(1, kv, 1, group, 1) * away[:, None, :, None]
    x = x.masked_fill_(~seen[:, None, :, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    del x
    z = p.sum(-1, keepdim=True)
    lse = (m + torch.log(z)).squeeze(-1)
    p /= torch.where(z == 0, 1.0, z)
    o = torch.matmul(p.reshape(seqs, kv, -1, tokens), v).reshape(*p.shape[:-1], c["dim"])
    back = lambda y: y.transpose(1, 2).flatten(2, 3)[b, i]  # noqa: E731
    return back(o).to(q.dtype), back(lse)


def _plain_accept(s, lengths):
    """(path, count, next token); the accepted rows moved, lengths cut."""
    c = s["case"]
    seqs, new = c["seqs"], c["new"]
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(seqs + 1, device=DEV) * new
    b, _ = _new_tokens(s)
    i = torch.arange(s["tokens"], device=DEV) - cu[b]
    there = cu[1:] - cu[:-1]
    pad = lambda x, fill: torch.full((seqs, new), fill, dtype=x.dtype, device=DEV).index_put_((b, i), x)  # noqa: E731
    tree, drafts, sampled = pad(s["tree"], 0), pad(s["drafts"], -1), pad(s["sampled"], -2)
    j = torch.arange(new, device=DEV)
    bit = torch.ones((), dtype=torch.int64, device=DEV) << j
    at = torch.zeros(seqs, dtype=torch.int64, device=DEV)
    path = torch.full((seqs, new), -1, dtype=torch.int64, device=DEV)
    path[:, 0] = torch.where(there > 0, 0, -1)
    alive = there > 0
    for step in range(1, new):
        child = (tree == (tree.gather(1, at[:, None]) | bit)) & (drafts == sampled.gather(1, at[:, None]))
        child &= (j > at[:, None]) & (j < there[:, None]) & alive[:, None]
        found = torch.where(child, j, new).amin(-1)
        alive = found < new
        path[:, step] = torch.where(alive, found, -1)
        at = torch.where(alive, found, at)
    count = (path >= 0).sum(-1)
    # rows that are not moved are put where they are
    base = s["lengths"].long() - there
    size = s["codes"].shape[3]
    where = path[b, i]
    page, slot = _slot(s["table"], size, b, base[b] + torch.where(where >= 0, where, i))
    to, at_slot = _slot(s["table"], size, b, base[b] + i)
    for x in (0, 1):
        s["codes"][x][to, :, at_slot] = s["codes"][x][page, :, slot]
        s["scales"][x][to, :, at_slot] = s["scales"][x][page, :, slot]
    lengths.sub_((there - count).int())
    token = torch.where(there > 0, sampled.gather(1, at[:, None]).squeeze(1), -1)
    return where.int(), count.int(), token


def _plain_sample(s):
    x, v = s["logits"].double(), s["case"]["vocab"]
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    index = torch.arange(v, device=DEV)
    first = torch.where(x == top, index, v).amin(-1)
    t = s["temperature"].double()[:, None] if s["temperature"] is not None else torch.ones_like(top)
    greedy = ~(t > 0)
    d = torch.where(x == top, 0.0, (x - top) / torch.where(greedy, 1.0, t))
    w = torch.round(torch.exp(d) * UNIT).long()
    del d
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    del x
    w = w.gather(-1, order)
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep &= (index < k) | (k <= 0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        inside = torch.where(keep, w, 0)
        before = inside.cumsum(-1) - inside
        keep &= (before.double() < p * inside.sum(-1, keepdim=True).double()) | (index == 0) | ~(p < 1)
    if s["min_p"] is not None:
        keep &= w.double() >= s["min_p"].double()[:, None] * UNIT
    w = torch.zeros_like(w).scatter_(-1, order, torch.where(keep, w, 0))
    sums = w.cumsum(-1)
    total = sums[:, -1]
    r = torch.minimum(torch.floor(s["random"].double() * total.double()).long(), total - 1)
    token = (sums <= r[:, None]).sum(-1)
    chance = torch.log(w.gather(-1, token[:, None]).squeeze(-1).double() / total.double())
    none = top[:, 0] == -math.inf
    token = torch.where(none, -1, torch.where(greedy[:, 0], first, token))
    return token, torch.where(none, -math.inf, torch.where(greedy[:, 0], 0.0, chance)).float()


def run(s):
    c = s["case"]
    kind, o = c["kind"], _ops() if own else None
    if kind == "sample":
        if own:
            return o.sample_tokens(s["logits"], s["random"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        return _plain_sample(s)
    if kind == "pages":
        now = s["now"]
        torch._foreach_copy_(list(now.values()), list(s["first"].values()))
        if own:
            made = o.kv4_reserve(s["new"], now["lengths"], now["table"], now["free"], now["count"], c["page"], s["n"])
        else:
            made = _plain_pages(s)
        return (*made, now["lengths"], now["table"], now["free"], now["count"])
    if kind == "rotate":
        if own:
            out = o.rotary(s["x"], s["positions"], s["freqs"], interleaved=c["interleaved"])
            return out, torch.autograd.grad(out, s["x"], s["grad"])[0]
        return (_turn(s["x"].detach(), s["positions"], s["freqs"], c["interleaved"]),
                _turn(s["grad"], s["positions"], s["freqs"], c["interleaved"], True))
    q, key, value = _parts(s)
    codes, scales, lengths, cu, table = s["codes"], s["scales"], s["lengths"], s["cu"], s["table"]
    if kind == "tree":
        if own:
            return o.kv4_tree_attention(q, codes, scales, lengths, s["tree"], cu, c["new"] if cu is not None else None,
                                        table, scale=s["scale"], softcap=c["softcap"], window=c["window"],
                                        slopes=s["slopes"])
        return _plain_tree(s)
    if kind == "place":
        if own:
            q = o.kv4_append_rotary(q, key, value, codes, scales, lengths, s["freqs"], cu, table, s["positions"],
                                    interleaved=c["interleaved"])
            return (q, *o.kv4_read(codes, scales, lengths, key.shape[0], cu, table, key.dtype))
        pos = s["positions"] if s["positions"] is not None else _new_tokens(s)[1]
        page, slot = _write(s, _turn(key, pos, s["freqs"], c["interleaved"]), value)
        return (_turn(q, pos, s["freqs"], c["interleaved"]), *_read(s, page, slot, key.dtype))
    cut = lengths.clone()
    if own:
        o.kv4_append(key, value, codes, scales, lengths, cu, table)
        made = o.kv4_accept(s["tree"], s["drafts"], s["sampled"], codes, scales, cut, cu, table)
        return (*made, cut, *o.kv4_read(codes, scales, lengths, key.shape[0], cu, table, key.dtype))
    page, slot = _write(s, key, value)
    made = _plain_accept(s, cut)
    return (*made, cut, *_read(s, page, slot, key.dtype))


# ---------------------------------------------------------------------------
# in 64 bits, one sequence and head at a time
# ---------------------------------------------------------------------------
def _exact_held(x):
    """What the cache holds of x [..., D], in 64 bits."""
    level = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    b = x.double().unflatten(-1, (-1, BLOCK))
    t = torch.float32 if x.dtype == torch.float16 else x.dtype
    e = torch.log2(b.abs().amax(-1, keepdim=True)).to(t).double().floor() - 2
    v = torch.ldexp(b, -e).to(torch.bfloat16).double()
    far = (v.abs()[..., None] - level).abs()
    # of two levels as near, the one with the even code
    pick = (far + 1e-12 * (torch.arange(8, device=x.device) % 2)).argmin(-1)
    return torch.ldexp(torch.copysign(level[pick], v), e).flatten(-2)


def _exact_values(codes, scales):
    """[tokens, D] in 64 bits from codes [tokens, D / 2] and scales: a code is
    sign, two exponent bits and one of the fraction."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    sign = torch.where(c >= 8, -1.0, 1.0)
    m = c % 8
    e = torch.div(m, 2, rounding_mode="floor")
    f = m % 2
    level = torch.where(e == 0, f / 2, torch.pow(2.0, e - 1) * (1 + f / 2))
    x = torch.ldexp(torch.ones((), dtype=torch.float64, device=codes.device), scales.double() - 127)
    return sign * level * x.repeat_interleave(BLOCK, -1)


def _exact_turn(x, positions, freqs, interleaved):
    """x as complex numbers times exp(i angle), in 64 bits, not rounded."""
    r = 2 * freqs.shape[0]
    y = x.double().clone()
    angle = torch.outer(positions.double(), freqs.double())
    z = torch.polar(torch.ones_like(angle), torch.remainder(angle, 2 * math.pi))[:, None]
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    w = torch.complex(y[..., first], y[..., second]) * z
    y[..., first], y[..., second] = w.real, w.imag
    return y


def _host_spans(s):
    c = s["case"]
    cu = s["cu"].tolist() if s["cu"] is not None else [i * c["new"] for i in range(c["seqs"] + 1)]
    return list(zip(cu[:-1], cu[1:]))


def _exact_tree(s):
    c = s["case"]
    q = _parts(s)[0].double()
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    group = c["heads"] // c["kv"]
    masks = [m % (1 << 64) for m in s["tree"].tolist()]
    for b, (first, end) in enumerate(_host_spans(s)):
        n = int(s["lengths"][b])
        base = n - (end - first)
        away = torch.full((end - first, n), -1, dtype=torch.int64)
        for i in range(end - first):
            line = [j for j in range(end - first) if masks[first + i] >> j & 1]
            away[i, :base] = base + len(line) - 1 - torch.arange(base)
            for back, j in enumerate(reversed(line)):
                away[i, base + j] = back
        away = away.to(DEV)
        seen = (away >= 0) & ((away < c["window"]) if c["window"] else True)
        t = torch.arange(n, device=DEV)
        page, slot = _slot(s["table"], s["codes"].shape[3], torch.tensor(b, device=DEV), t)
        for h in range(c["kv"]):
            k, v = (_exact_values(s["codes"][i][page, h, slot], s["scales"][i][page, h, slot]) for i in (0, 1))
            for x in range(h * group, (h + 1) * group):
                a = q[first:end, x] @ k.T * s["scale"]
                if c["softcap"]:
                    a = c["softcap"] * torch.tanh(a / c["softcap"])
                if s["slopes"] is not None:
                    a = a - s["slopes"][x].double() * away
                a = a.masked_fill(~seen, -math.inf)
                z = torch.logsumexp(a, -1)
                out[first:end, x], lse[first:end, x] = torch.exp(a - z[:, None]) @ v, z
    return out, lse


def _exact_pages(s):
    c = s["case"]
    first = {k: v.tolist() for k, v in s["first"].items()}
    lengths, table, new = first["lengths"], first["table"], s["new"].tolist()
    room, stack, rest = len(first["free"]), first["free"][:first["count"][0]], first["free"]
    for b in range(c["seqs"]):
        if new[b] < 0:
            stack += [p for p in table[b] if 0 <= p < room]
            table[b], lengths[b] = [-1] * c["per"], 0
    rest = stack + rest[len(stack):]
    stock, wanted, tokens, top = len(stack), 0, 0, len(stack)
    cu, positions, slots = [0], [], []
    for b in range(c["seqs"]):
        grow = max(new[b], 0)
        if lengths[b] + grow <= c["per"] * c["page"]:
            places = range(lengths[b], lengths[b] + grow)
            lack = sorted({t // c["page"] for t in places if not 0 <= table[b][t // c["page"]] < room})
            wanted += len(lack)
            tokens += grow
            if (not lack or wanted <= stock) and tokens <= s["n"]:
                for j in lack:
                    top -= 1
                    table[b][j] = rest[top]
                for t in places:
                    positions.append(t)
                    slots.append(table[b][t // c["page"]] * c["page"] + t % c["page"])
                lengths[b] += grow
        cu.append(len(positions))
    left = [-1] * (s["n"] - len(positions))
    return tuple(torch.tensor(x) for x in (cu, positions + left, slots + left, lengths, table, rest, [top]))


def _exact_accept(s, key, value):
    held = [_exact_held(x) for x in (key, value)]
    masks = [m % (1 << 64) for m in s["tree"].tolist()]
    drafts, sampled = s["drafts"].tolist(), s["sampled"].tolist()
    lengths = s["lengths"].tolist()
    path, count, token, order = [], [], [], []
    for b, (first, end) in enumerate(_host_spans(s)):
        line = [0]
        while True:
            at = first + line[-1]
            child = [j for j in range(line[-1] + 1, end - first)
                     if masks[first + j] == masks[at] | 1 << j and drafts[first + j] == sampled[at]]
            if not child:
                break
            line.append(child[0])
        path += line + [-1] * (end - first - len(line))
        order += [first + j for j in line] + list(range(first + len(line), end))
        count.append(len(line))
        token.append(sampled[first + line[-1]])
        lengths[b] -= end - first - len(line)
    return (*(torch.tensor(x) for x in (path, count, token, lengths)), held[0][order], held[1][order])


def _exact_sample(s):
    """One row at a time, from its likeliest token down."""
    found, chance = [], []
    for r in range(s["case"]["rows"]):
        x = s["logits"][r].double()
        value, order = torch.sort(x, descending=True, stable=True)
        t = float(s["temperature"][r]) if s["temperature"] is not None else 1.0
        if t <= 0:
            found.append(order[0])
            chance.append(torch.zeros_like(value[0]))
            continue
        p = torch.exp((value - value[0]) / t)
        m = x.shape[0]
        if s["top_k"] is not None:
            m = min(m, int(s["top_k"][r]))
        if s["top_p"] is not None and float(s["top_p"][r]) < 1:
            sums = p[:m].cumsum(0)
            m = min(m, 1 + int((sums[:-1] < float(s["top_p"][r]) * sums[-1]).sum()))
        if s["min_p"] is not None:
            m = min(m, int((p >= float(s["min_p"][r])).sum()))
        kept, rank = torch.sort(order[:m])
        sums = p[:m][rank].cumsum(0)
        at = min(m - 1, int((sums <= float(s["random"][r]) * sums[-1]).sum()))
        found.append(kept[at])
        chance.append(torch.log(p[rank[at]] / sums[-1]))
    return torch.stack(found), torch.stack(chance)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "sample":
        return _exact_sample(s)
    if kind == "pages":
        return _exact_pages(s)
    if kind == "tree":
        return _exact_tree(s)
    if kind == "rotate":
        return (_exact_turn(s["x"].detach(), s["positions"], s["freqs"], case["interleaved"]),
                _exact_turn(s["grad"], -s["positions"], s["freqs"], case["interleaved"]))
    q, key, value = _parts(s)
    if kind == "accept":
        return _exact_accept(s, key, value)
    pos = s["positions"]
    if pos is None:
        pos = torch.cat([torch.arange(int(n) - (end - first), int(n), device=DEV)
                         for n, (first, end) in zip(s["lengths"], _host_spans(s))])
    key = _exact_turn(key, pos, s["freqs"], case["interleaved"]).to(key.dtype)
    return _exact_turn(q, pos, s["freqs"], case["interleaved"]), _exact_held(key), _exact_held(value)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "sample":
        size = torch.finfo(TYPES[c["type"]]).bits // 8
        # a subtraction, a product, an exponential and a sum for each token
        return {"bytes": c["rows"] * (c["vocab"] * size + 32), "flops": 4 * c["rows"] * c["vocab"]}
    if c["kind"] == "pages":
        lens, new = _page_sizes(c)
        n = int(new.clamp(min=0).sum())
        touched = int((-(-(lens + new.clamp(min=0)) // c["page"]) - lens // c["page"]).sum())
        ended = int((new < 0).sum()) * c["per"]
        # new, lengths in and out, offsets; table entries and free pages; positions and slots
        return {"bytes": 16 * c["seqs"] + 12 * (touched + ended) + 12 * n, "flops": 0}
    lens, new = _sizes(c)
    n, size = int(new.sum()), torch.finfo(TYPES[c["type"]]).bits // 8
    token = c["kv"] * c["dim"] * 17 // 32  # bytes of a token's keys, or values
    row = c["dim"] * size
    if c["kind"] == "rotate":
        return {"bytes": 4 * n * c["heads"] * row + 4 * n, "flops": 2 * 3 * n * c["heads"] * c["turned"]}
    if c["kind"] == "place":
        # queries in and out, keys and values in, codes out and in again, values out
        return {"bytes": 2 * n * c["heads"] * row + 4 * n * c["kv"] * row + 4 * n * token,
                "flops": 3 * n * (c["heads"] + c["kv"]) * c["turned"]}
    if c["kind"] == "accept":
        # keys and values in, codes out and in again, values out; masks, drafted and sampled tokens
        return {"bytes": 4 * n * c["kv"] * row + 4 * n * token + 28 * n, "flops": 0}
    seen = keys = 0
    for length, t in zip(lens.tolist(), new.tolist()):
        w = c["window"] or length
        seen += t * min(w, length - t // 2)
        keys += min(length, t + w - 1)
    return {"bytes": 2 * token * keys + 2 * n * c["heads"] * row + 4 * n * c["heads"] + 8 * n,
            "flops": 4 * c["dim"] * c["heads"] * seen}
