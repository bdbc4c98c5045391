"""Plain 64-bit forms of the 4-bit cache's operators, on the CPU, for their tests."""

import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def decode(codes, scales):
    """Values of codes [..., D / 2] and scale bytes [..., D / 32]; 255 is NaN."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = torch.where(c >= 8, -1.0, 1.0).double() * LEVELS[c % 8]
    s = torch.ldexp(torch.ones((), dtype=torch.float64), scales.double() - 127)
    s = torch.where(scales == 255, math.nan, s)
    return v * s.repeat_interleave(32, -1)


def quantize(x):
    """Codes and scale bytes of finite x [..., D]: the scale is 2 ** (floor(log2
    of the block's largest magnitude) - 2) within E8M0, the log in x's type (fp32
    for fp16), and a quotient, as bf16, goes to the nearest level, ties to the
    even code, zeros to code 0."""
    b = x.double().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    log = torch.log2(torch.where(amax == 0, 2.0 ** -126, amax).to(torch.float32 if x.dtype == torch.float16 else x.dtype))
    e = (log.double().floor() - 2).clamp(-127, 127)
    v = torch.ldexp(b, -e).to(torch.bfloat16).double()
    far = (v.abs()[..., None] - LEVELS).abs() + 1e-9 * (torch.arange(8) % 2)  # of two as near, the even code
    code = (far.argmin(-1) + 8 * ((v < 0) | ((v == 0) & (b < 0)))).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, (e + 127).squeeze(-1).to(torch.uint8)


def places(table, size, pages, b, tokens):
    """[(token, page, slot)] of sequence b's tokens that have a page."""
    found = []
    for t in tokens:
        page = b if table is None else int(table[b, t // size])
        if 0 <= page < pages:
            found.append((t, page, t if table is None else t % size))
    return found


def room(codes, table):
    return codes.shape[3] * (1 if table is None else table.shape[1])


def spans(n, seqs, cu):
    cu = cu.tolist() if cu is not None else [i * (n // seqs) for i in range(seqs + 1)]
    return list(zip(cu[:-1], cu[1:]))


def attention(q, codes, scales, lengths, cu=None, table=None, scale=None, softcap=0.0, window=0, slopes=None):
    """(out, lse, weights {(b, kv head): [tokens]}, size [N, H, D] of what an
    output sums, error [N, H]: how far a score may be off in fp32 and with
    queries held to 2^-22 of their largest)."""
    n, heads, dim = q.shape
    pages, kv, size = codes.shape[1:4]
    seqs, group = lengths.shape[0], heads // kv
    scale = dim ** -0.5 if scale is None else scale
    q = q.double()
    out, mass = torch.zeros(n, heads, dim, dtype=torch.float64), torch.zeros(n, heads, dim, dtype=torch.float64)
    lse, err = torch.full((n, heads), -math.inf, dtype=torch.float64), torch.zeros(n, heads, dtype=torch.float64)
    added = torch.zeros(seqs, kv, room(codes, table), dtype=torch.float64)
    for b, (first, end) in enumerate(spans(n, seqs, cu)):
        length = int(lengths[b])
        where = places(table, size, pages, b, range(max(0, min(length, room(codes, table)))))
        if not where:
            continue
        t, page, slot = (torch.tensor(x) for x in zip(*where))
        for h in range(kv):
            k, v = (decode(codes[i][page, h, slot], scales[i][page, h, slot]) for i in (0, 1))
            for i in range(first, end):
                away = length - (end - i) - t
                seen = (away >= 0) & ((away < window) if window else True)
                if not bool(seen.any()):
                    continue
                for x in range(h * group, (h + 1) * group):
                    a = k[seen] @ q[i, x] * scale
                    if softcap:
                        a = softcap * torch.tanh(a / softcap)
                    if slopes is not None:
                        a = a - slopes[x].double() * away[seen]
                    z = torch.logsumexp(a, 0)
                    p = torch.exp(a - z)
                    out[i, x], lse[i, x] = p @ v[seen], z
                    # a NaN value matters to the rows that see it, also at weight 0
                    mass[i, x] = p @ v[seen].abs().nan_to_num()
                    added[b, h, t[seen]] += p
                    big = (k[seen].abs() @ q[i, x].abs()).nan_to_num().max()
                    err[i, x] = abs(scale) * ((dim + 4) * 2.0 ** -24 * big
                                              + 2.0 ** -22 * q[i, x].abs().max() * k[seen].abs().sum(-1).nan_to_num().max())
                    # the score's own roundings: times scale and log2 e, capped, sloped
                    err[i, x] += 8 * 2.0 ** -24 * (a.abs().nan_to_num().max() + softcap)
                    if slopes is not None:
                        err[i, x] += 4 * 2.0 ** -24 * (slopes[x].abs() * away[seen].max())
    return out, lse, added, mass, err


def kept(weights, lengths, budget, recent):
    """(index [B, kv, budget], new lengths, weights kept)."""
    seqs, kv, most = weights.shape
    index = torch.full((seqs, kv, budget), -1, dtype=torch.int32)
    w = torch.zeros(seqs, kv, budget)
    lens = []
    for b in range(seqs):
        n = min(max(int(lengths[b]), 0), most)
        old = max(0, n - recent)
        lens.append(min(n, budget))
        for h in range(kv):
            x = weights[b, h].tolist()
            heavy = sorted(range(old), key=lambda i: (0 if math.isnan(x[i]) else 1, -x[i] if x[i] == x[i] else 0.0, i))
            keep = sorted(heavy[:min(n, budget) - (n - old)]) + list(range(old, n))
            index[b, h, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
            w[b, h, :len(keep)] = weights[b, h, keep]
    return index, torch.tensor(lens, dtype=torch.int32), w
