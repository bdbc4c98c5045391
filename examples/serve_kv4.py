"""Serve a batch of prompts from a 4-bit cache of keys and values.

    python3 examples/serve_kv4.py [--seqs 4] [--prompt 1500] [--budget 512] [--steps 32]

One attention layer with random weights, as a server runs it:

1. admission: the prompts' keys and values are appended to a paged cache
   (``kv4_append``), every prompt token attends to what is before it
   (``kv4_attention``), and the last tokens of each prompt say which of its
   tokens matter (``kv4_accumulate``);
2. each sequence is cut down to a budget, the heaviest tokens and the latest
   ones, in the cache that decoding reads (``kv4_evict``);
3. a decode step (append, attend, weigh) is captured into a graph once and
   replayed as the sequences grow.

It prints how far the attention over the 4-bit cache is from one over the keys
and values that were appended, and what the caches take.
"""

import argparse
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import __graft_entry__  # noqa: E402


def pages(tokens, seqs, kv, dim, page, device):
    """(codes, scales, table) of an empty cache with room for `tokens` each."""
    each = -(-tokens // page)
    table = torch.randperm(seqs * each, device=device).int().reshape(seqs, each)
    codes = torch.zeros(2, seqs * each, kv, page, dim // 2, dtype=torch.uint8, device=device)
    scales = torch.zeros(2, seqs * each, kv, page, dim // 32, dtype=torch.uint8, device=device)
    return codes, scales, table


class Layer:
    """Queries, keys and values of one attention layer from one projection."""

    def __init__(self, width, heads, kv, dim, device):
        self.heads, self.kv, self.dim = heads, kv, dim
        g = torch.Generator(device).manual_seed(0)
        self.weight = torch.randn((heads + 2 * kv) * dim, width, device=device, generator=g).mul_(width ** -0.5).bfloat16()

    def __call__(self, x):
        y = torch.nn.functional.linear(x, self.weight).reshape(x.shape[0], -1, self.dim)
        return y.split([self.heads, self.kv, self.kv], 1)


def plain(q, k, v):
    """Causal attention of one sequence in fp32, for comparison."""
    group = q.shape[1] // k.shape[1]
    q, k, v = (t.float().transpose(0, 1) for t in (q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)))
    s = torch.matmul(q, k.transpose(1, 2).contiguous()) * q.shape[-1] ** -0.5
    s = s.masked_fill(torch.ones_like(s[0], dtype=torch.bool).triu(1), -math.inf)
    return torch.matmul(torch.softmax(s, -1), v).transpose(0, 1)


def serve(seqs=4, prompt=1500, budget=512, steps=32, heads=16, kv=4, dim=128, width=1024, page=64, recent=64,
          device="cuda"):
    __graft_entry__.load_package()
    ops = torch.ops.quantized_ops
    torch.manual_seed(0)
    layer = Layer(width, heads, kv, dim, device)
    news = [prompt - prompt * i // (2 * seqs) for i in range(seqs)]  # ragged prompts
    cu = torch.tensor([0] + news, device=device).cumsum(0).int()
    lengths = torch.tensor(news, device=device).int()

    # 1. admission
    codes, scales, table = pages(prompt, seqs, kv, dim, page, device)
    q, k, v = layer(torch.randn(sum(news), width, device=device).bfloat16())
    ops.kv4_append(k, v, codes, scales, lengths, cu, table)
    out, lse = ops.kv4_attention(q, codes, scales, lengths, cu, prompt, table)
    want = plain(q[:news[0]], k[:news[0]], v[:news[0]])
    error = float((out[:news[0]].float() - want).norm() / want.norm())
    last = min(recent, min(news))  # the queries that say what matters
    tail = torch.cat([torch.arange(int(e) - last, int(e), device=device) for e in cu[1:]])
    weights = torch.zeros(seqs, kv, prompt, device=device)
    ops.kv4_accumulate(q[tail], lse[tail], codes, scales, lengths, weights, None, None, table)

    # 2. the cache that decoding reads: the budget and room for the steps
    small = pages(budget + steps, seqs, kv, dim, page, device)
    small_weights = torch.zeros(seqs, kv, budget, device=device)
    index, kept = ops.kv4_evict(codes, scales, weights, lengths, budget, recent, small[0], small[1], small_weights,
                                table, small[2])
    weights = torch.zeros(seqs, kv, budget + steps, device=device)
    weights[..., :budget] = small_weights

    # 3. decoding
    x = torch.randn(seqs, width, device=device).bfloat16()

    def step():
        kept.add_(1)
        q, k, v = layer(x)
        ops.kv4_append(k, v, small[0], small[1], kept, None, small[2])
        out, lse = ops.kv4_attention(q, small[0], small[1], kept, None, None, small[2])
        ops.kv4_accumulate(q, lse, small[0], small[1], kept, weights, None, None, small[2])
        return out

    before = kept.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # warm: what the capture calls is loaded
    torch.cuda.current_stream().wait_stream(side)
    kept.copy_(before)
    weights[..., :budget] = small_weights
    weights[..., budget:] = 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    outputs = []
    for _ in range(steps):
        x.copy_(torch.randn(seqs, width, device=device))
        graph.replay()
        outputs.append(out.clone())
    torch.cuda.synchronize()
    size = lambda c: (c[0].numel() + c[1].numel()) / 2 ** 20  # noqa: E731
    return dict(error=error, kept=kept.tolist(), index=index, weights=weights, outputs=torch.stack(outputs),
                prompt_mib=size((codes, scales)), decode_mib=size(small))


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("seqs", 4), ("prompt", 1500), ("budget", 512), ("steps", 32)):
        p.add_argument(f"--{name}", type=int, default=value)
    r = serve(**vars(p.parse_args()))
    print(f"attention of the first prompt: off by {r['error']:.3f} of its norm (keys and values in 4 bits)")
    print(f"cache of the prompts {r['prompt_mib']:.2f} MiB, of decoding {r['decode_mib']:.2f} MiB")
    print(f"tokens kept and decoded: {r['kept']}; outputs {list(r['outputs'].shape)}, "
          f"all finite: {bool(r['outputs'].isfinite().all())}")


if __name__ == "__main__":
    main()
