"""Decode from a 4-bit cache with drafted tokens.

    python3 examples/draft_kv4.py [--seqs 4] [--prompt 200] [--new 64] [--temperature 0.8] [--plain]

One layer with random weights, as a server decodes with it:

1. admission: ``kv4_reserve`` hands out pages for the prompts, their queries and
   keys are turned to their positions on the way into the cache
   (``kv4_append_rotary``), every prompt token attends to what is before it
   (``kv4_attention``) and the first new token is drawn (``sample_tokens``);
2. a step: a small tree of tokens that may come next is drafted from each
   sequence's last token, appended, attended to as a tree (``kv4_tree_attention``),
   a token is drawn after each of its nodes, and those drafted tokens that were
   drawn are kept (``kv4_accept``).  The step is captured into a graph once and
   replayed; lengths, pages and tokens stay on the device.

A token is drawn with the random number of its sequence and place, so that with
drafts (the default) and without (--plain) the same tokens come out, but for the
rounding of their logits, in fewer steps with them.
"""

import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import __graft_entry__  # noqa: E402

PARENTS = [-1, 0, 0, 1, 1, 2, 3, 6]  # of the drafted tree's nodes; node 0 is the token known already
RANKS = [0, 0, 1, 0, 1, 0, 0, 0]     # which of its parent's likely successors each is


class Model:
    """Embeddings, one attention layer and logits by the embeddings again."""

    def __init__(self, vocab, width, heads, kv, dim, device):
        self.heads, self.kv, self.dim = heads, kv, dim
        g = torch.Generator(device).manual_seed(0)
        rand = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
        self.embed = rand(vocab, width)
        self.project = rand((heads + 2 * kv) * dim, width) * width ** -0.5
        self.mix = rand(width, heads * dim) * (2.0 / (heads * dim)) ** 0.5
        # what a token alone makes likely: the drafts
        self.likely = self.logits(self.embed, torch.zeros(vocab, heads, dim, device=device)).topk(2).indices

    def qkv(self, x):
        y = torch.nn.functional.linear(x, self.project).reshape(x.shape[0], -1, self.dim)
        return y.split([self.heads, self.kv, self.kv], 1)

    def logits(self, x, attended):
        h = torch.nn.functional.linear(attended.flatten(1), self.mix) + torch.roll(x, 1, -1)
        return torch.nn.functional.linear(h, self.embed) * (4.0 / self.embed.shape[1] ** 0.5)


def tree_of(parents):
    """(ancestors of each node as bits, itself included; its depth)."""
    masks = [1]
    for j in range(1, len(parents)):
        masks.append(masks[parents[j]] | 1 << j)
    return masks, [bin(m).count("1") - 1 for m in masks]


def generate(seqs=4, prompt=200, new=64, temperature=0.8, drafted=True, top_k=20, top_p=0.95, vocab=512, width=256,
             heads=8, kv=2, dim=64, page=16, device="cuda"):
    vqx = __graft_entry__.load_package()
    ops = torch.ops.quantized_ops
    torch.manual_seed(1)
    model = Model(vocab, width, heads, kv, dim, device)
    freqs = vqx.ops.rotary_frequencies(dim, device=device)
    parents, ranks = (PARENTS, RANKS) if drafted else (PARENTS[:1], RANKS[:1])
    masks, depth = tree_of(parents)
    nodes, room = len(parents), prompt + new + len(PARENTS)
    i32 = lambda *a, **k: torch.zeros(*a, dtype=torch.int32, device=device, **k)  # noqa: E731

    # an empty cache and its pages
    each = -(-room // page)
    codes = torch.zeros(2, seqs * each, kv, page, dim // 2, dtype=torch.uint8, device=device)
    scales = torch.zeros(2, seqs * each, kv, page, dim // 32, dtype=torch.uint8, device=device)
    lengths, table = i32(seqs), i32(seqs, each) - 1
    free, count = torch.randperm(seqs * each, device=device).int(), i32(1) + seqs * each

    # how tokens are drawn, the same for a place however it is come to
    random = torch.rand(seqs, room + 1, device=device)
    said = torch.full((seqs, room + 1), -1, dtype=torch.int64, device=device)

    def draw(logits, rows, places):
        f = lambda v, t: torch.full((rows.shape[0],), v, dtype=t, device=device)  # noqa: E731
        return ops.sample_tokens(logits, random[rows, places + 1], f(temperature, torch.float32), f(top_k, torch.int32),
                                 f(top_p, torch.float32))[0]

    # 1. admission of ragged prompts
    news = [prompt - prompt * i // (2 * seqs) for i in range(seqs)]
    cu, places, _ = ops.kv4_reserve(torch.tensor(news, device=device).int(), lengths, table, free, count, page, sum(news))
    x = model.embed[torch.randint(vocab, (sum(news),), device=device)]
    q = ops.kv4_append_rotary(*model.qkv(x), codes, scales, lengths, freqs, cu, table)
    out, _ = ops.kv4_attention(q, codes, scales, lengths, cu, prompt, table)
    last, rows = cu[1:].long() - 1, torch.arange(seqs, device=device)
    token = draw(model.logits(x[last], out[last]), rows, places[last].long())
    said[rows, lengths.long()] = token

    # 2. decoding
    grow = i32(seqs) + nodes
    tree = torch.tensor(masks * seqs, device=device)
    rows = rows.repeat_interleave(nodes)
    # a node's position is as far behind the cached tokens as it has ancestors
    behind = (torch.tensor(depth) - torch.arange(nodes)).int().repeat(seqs).to(device)
    kept, limit = i32(seqs), lengths + new

    def step():
        drafts = [token]
        for j in range(1, nodes):
            drafts.append(model.likely[drafts[parents[j]], ranks[j]])
        ids = torch.stack(drafts, 1).flatten()
        cu, places, _ = ops.kv4_reserve(grow, lengths, table, free, count, page, seqs * nodes)
        positions = places + behind
        x = model.embed[ids]
        q = ops.kv4_append_rotary(*model.qkv(x), codes, scales, lengths, freqs, cu, table, positions)
        out, _ = ops.kv4_tree_attention(q, codes, scales, lengths, tree, cu, nodes, table)
        sampled = draw(model.logits(x, out), rows, positions.long().clamp(max=room - 1))
        path, accepted, follows = ops.kv4_accept(tree, ids, sampled, codes, scales, lengths, cu, table)
        # what was drawn after each accepted node is said at the next place
        at = (path.reshape(seqs, nodes).long() + nodes * torch.arange(seqs, device=device)[:, None]).clamp(min=0)
        place = torch.where(path.reshape(seqs, nodes) >= 0, positions[at].long() + 1, room).clamp(max=room)
        said.scatter_(1, place, sampled[at])
        token.copy_(follows)
        kept.copy_(accepted)
        torch.minimum(lengths, limit, out=lengths)  # a sequence that has all of its tokens stays there

    state = [codes, scales, lengths, table, free, count, token, said, kept]
    before = [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # warm: what the capture calls is loaded
    torch.cuda.current_stream().wait_stream(side)
    for t, b in zip(state, before):
        t.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    steps, line = 0, []
    while bool((lengths < limit).any()):
        graph.replay()
        steps += 1
        line.append(kept.clone())
    torch.cuda.synchronize()
    tokens = [said[b, n:n + new].tolist() for b, n in enumerate(news)]
    return dict(tokens=tokens, steps=steps, accepted=torch.stack(line).float().mean().item(), lengths=lengths.tolist(),
                table=table, free=free, count=int(count))


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("seqs", 4), ("prompt", 200), ("new", 64), ("temperature", 0.8)):
        p.add_argument(f"--{name}", type=type(value), default=value)
    p.add_argument("--plain", action="store_true", help="without drafts")
    a = p.parse_args()
    r = generate(a.seqs, a.prompt, a.new, a.temperature, drafted=not a.plain)
    print(f"{r['steps']} steps, {r['accepted']:.2f} tokens a step and sequence; lengths {r['lengths']}")
    print("first tokens:", [t[:8] for t in r["tokens"]])


if __name__ == "__main__":
    main()
