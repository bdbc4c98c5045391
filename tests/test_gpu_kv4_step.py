"""A server's step of drafted tokens, its operators one after the other: pages are
reserved, keys turned and appended, the tree is attended to, tokens are drawn and
accepted.  Some steps of it, called and captured, against lists and 64-bit forms."""

import importlib.util
import os
import random

import pytest
import torch

from tests import kv4_reference as ref
from tests.test_gpu_kv4 import same
from tests.test_gpu_kv4_pages import accepted, forest, reserved, signed
from tests.test_gpu_kv4_tree import TYPES, check
from tests.test_gpu_rotary import turned
from tests.test_gpu_sampling import sampled

pytestmark = pytest.mark.gpu

DEV = "cuda"


class Server:
    """The device's state and its step, and the same in lists."""

    def __init__(self, vqx, kind, seqs, kv, group, dim, page, per, pages, n, interleaved):
        self.ops, self.kind, self.page, self.n, self.interleaved = torch.ops.quantized_ops, kind, page, n, interleaved
        z = lambda *s, t=torch.int32: torch.zeros(*s, dtype=t, device=DEV)  # noqa: E731
        self.codes, self.scales = z(2, pages, kv, page, dim // 2, t=torch.uint8), z(2, pages, kv, page, dim // 32, t=torch.uint8)
        self.lengths, self.table, self.count = z(seqs), z(seqs, per) - 1, z(1) + pages
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).int().to(DEV)
        self.grow, self.behind, self.tree = z(seqs), z(n), z(n, t=torch.int64)
        self.drafts, self.bias, self.random = z(n, t=torch.int64), z(n, 6, t=torch.float32), z(n, t=torch.float32)
        self.q, self.k, self.v = (z(n, h, dim, t=TYPES[kind]) for h in (kv * group, kv, kv))
        self.freqs = vqx.ops.rotary_frequencies(dim, device=DEV)
        # in lists
        self.state = ([0] * seqs, [[-1] * per for _ in range(seqs)], self.free.tolist(), pages)
        self.held = [[] for _ in range(seqs)]  # (codes, scales) of each token

    def step(self):
        made = self.ops.kv4_reserve(self.grow, self.lengths, self.table, self.free, self.count, self.page, self.n)
        positions = made[1] + self.behind
        q = self.ops.kv4_append_rotary(self.q, self.k, self.v, self.codes, self.scales, self.lengths, self.freqs, made[0],
                                       self.table, positions, interleaved=self.interleaved)
        out, lse = self.ops.kv4_tree_attention(q, self.codes, self.scales, self.lengths, self.tree, made[0], 25, self.table)
        logits = self.bias + out[:, 0, :6].float()
        tokens, chances = self.ops.sample_tokens(logits, self.random)
        before = self.codes.clone(), self.scales.clone(), self.lengths.clone()
        path, counts, follows = self.ops.kv4_accept(self.tree, self.drafts, tokens, self.codes, self.scales, self.lengths,
                                                    made[0], self.table)
        return *made, q, out, lse, logits, tokens, *before, path, counts, follows

    def inputs(self, grow, seed):
        g = torch.Generator().manual_seed(seed)
        # a server looks at what it was given: tokens of a sequence without pages wait
        cu = reserved(list(grow), list(self.state[0]), [list(x) for x in self.state[1]], list(self.state[2]), self.state[3],
                      self.page, self.n)[0]
        news = [end - first for first, end in zip(cu[:-1], cu[1:])]
        tree, drafts, say = forest(news, seed, likely=0.8)
        depth = [bin(m).count("1") - 1 for m in tree]
        at = [j for c in news for j in range(c)]
        rest = [0] * (self.n - len(tree))
        self.grow.copy_(torch.tensor(grow))
        self.tree.copy_(torch.tensor([signed(m) for m in tree] + rest))
        self.behind.copy_(torch.tensor([d - j for d, j in zip(depth, at)] + rest))
        self.drafts.copy_(torch.tensor(drafts + rest))
        self.bias.copy_(6.0 * torch.nn.functional.one_hot(torch.tensor(say + rest), 6))
        self.random.copy_(torch.rand(self.n, generator=g))
        for t in (self.q, self.k, self.v):
            t.copy_(torch.randn(t.shape, generator=g))
        self.host = grow, tree, drafts

    def check(self, made):
        """What a step made of the last inputs; the lists follow it."""
        grow, tree, drafts = self.host
        cu, places, slots, q, out, lse, logits, tokens, codes, scales, lengths, path, counts, follows = made
        ended = [b for b, x in enumerate(grow) if x < 0]
        want = reserved(grow, *self.state, self.page, self.n)
        for name, got, w in zip(("cu", "positions", "slots"), (cu, places, slots), want):
            same(got, torch.tensor(w, dtype=got.dtype), name)
        live, seqs = want[0][-1], len(grow)
        spans = list(zip(want[0][:-1], want[0][1:]))
        same(lengths, torch.tensor(want[3]).int(), "lengths before")

        # turned queries: those of the operator by itself
        positions = places + self.behind
        alone = self.ops.rotary(self.q, positions, self.freqs, interleaved=self.interleaved)
        same(q[:live], alone[:live].cpu(), "queries")
        keys = turned(self.k.cpu(), positions.cpu(), self.freqs.cpu(), self.interleaved).float().to(self.k.dtype)
        table = self.table.cpu()
        host = [t.cpu() for t in (q, codes, scales, lengths, cu)]
        again = check(self.ops, self.kind, *host[:4], tree + [0] * (self.n - len(tree)), host[4], 25, table, live)
        same(out[:live], again[0].cpu(), "out")
        same(lse[:live], again[1].cpu(), "lse")
        say = [sampled(row, float(u))[0] for row, u in zip(logits.double().tolist(), self.random.tolist())]
        assert tokens.tolist()[:live] == say[:live]

        line, kept, follow = accepted(tree[:live], drafts[:live], say[:live], spans)
        same(path[:live], torch.tensor(line).int(), "path")
        same(counts, torch.tensor(kept).int(), "accepted")
        same(follows, torch.tensor(follow), "next")
        for b, (first, end) in enumerate(spans):
            if b in ended:
                self.held[b] = []
            for i in range(kept[b]):
                row = first + line[first + i]
                self.held[b].append([torch.stack(x) for x in zip(ref.quantize(keys[row]), ref.quantize(self.v[row].cpu()))])
        left = [n - (end - first) + k for n, (first, end), k in zip(want[3], spans, kept)]
        self.state = (left, *want[4:6], want[6])
        same(self.lengths, torch.tensor(left).int(), "lengths")
        same(self.table, torch.tensor(want[4]).int(), "table")
        same(self.free, torch.tensor(want[5]).int(), "free")
        assert self.count.item() == want[6] and left == [len(x) for x in self.held]
        # the cache holds the accepted tokens, as if no others had been there
        after = self.codes.cpu(), self.scales.cpu()
        for b in range(seqs):
            for (_, p, s), token in zip(ref.places(table, self.page, after[0].shape[1], b, range(left[b])), self.held[b]):
                for got, w in zip(after, token):
                    same(got[:, p, :, s], w, f"token of sequence {b}")
        return kept


def growth(steps, seqs, most):
    """Prompts of one sequence after another, drafts of some nodes, ends."""
    r, lines, running = random.Random(seqs), [], [False] * seqs
    for i in range(steps):
        line = []
        for b in range(seqs):
            if not running[b] and r.random() < 0.6:
                line.append(r.randrange(1, most + 1))
                running[b] = True
            elif running[b] and r.random() < 0.15:
                line.append(-1)
                running[b] = False
            else:
                line.append(r.choice([0, 1, 2, 5, 9]) if running[b] else 0)
        lines.append(line)
    return lines


SERVERS = [
    # kind, seqs, kv, group, dim, page, pages per sequence, pages, new tokens at most, interleaved
    ("bf16", 3, 2, 4, 128, 16, 6, 5, 64, False),
    ("f32", 5, 1, 2, 64, 7, 9, 9, 90, True),
    ("f16", 2, 3, 1, 256, 32, 4, 2, 70, False),
]


@pytest.mark.parametrize("how", SERVERS)
@pytest.mark.parametrize("captured", [False, True])
def test_steps(vqx, how, captured):
    """Pages are few: where they run out, tokens wait."""
    server = Server(vqx, *how)
    step = server.step
    if captured:
        server.step()  # with grow of 0: nothing changes
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made = server.step()

        def step():
            graph.replay()
            return made

    total = 0
    for i, grow in enumerate(growth(12, how[1], 25)):
        server.inputs(grow, 100 + i)
        made = step()
        torch.cuda.synchronize()
        total += sum(server.check(made))
    assert total > 25


def test_the_drafting_example(vqx):
    """It runs, with drafts and without; every token asked for is there, pages are
    neither lost nor held twice."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "draft_kv4.py")
    spec = importlib.util.spec_from_file_location("draft_kv4", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    for drafted in (True, False):
        r = example.generate(seqs=3, prompt=50, new=20, drafted=drafted, vocab=200)
        assert r["lengths"] == [50 - 50 * b // 6 + 20 for b in range(3)]
        assert all(len(t) == 20 and all(0 <= x < 200 for x in t) for t in r["tokens"])
        held = r["table"][r["table"] >= 0].tolist() + r["free"][:r["count"]].tolist()
        assert sorted(held) == list(range(r["free"].shape[0]))
        assert r["steps"] <= 20 and (drafted or (r["steps"] == 20 and r["accepted"] == 1.0))
