"""One verify step of speculative decoding over drafted token trees, on the operators that stand between
the GEMVs:

    tree_layout -> rotary_append -> tree_attention -> lm_head (w8a16_gemv) -> sample_tokens -> accept

The model is a single attention layer with random weights, wide enough to run everything at its real
sizes; every step is captured in one CUDA graph, and replays follow the lengths and trees on the device.

    python examples/verify_step.py [--steps 8] [--context 4000] [--nodes 8]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import flash_next_rtxpro6000_b200 as fx  # noqa: E402


class VerifyStep:
    """The buffers of one request's verify step and the step itself.

    Node 0 of the tree is the last accepted token; the others are drafted.  After ``run`` the sampled
    token of every node is in ``sampled``; ``accept`` walks from node 0 along the drafted tokens that
    equal what was sampled at their parents, moves the accepted nodes' keys and values to the places
    after the context and returns the accepted tokens and the one sampled at the end."""

    def __init__(self, context: int, nodes: int, hidden: int = 2048, q_heads: int = 16, kv_heads: int = 2,
                 dim: int = 256, rotated: int = 64, vocab: int = 49152, page: int = 64, room: int = 1024,
                 temperature: float = 0.8, top_k: int = 50, top_p: float = 0.95, seed: int = 0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
        self.q_heads, self.kv_heads, self.dim, self.page, self.nodes = q_heads, kv_heads, dim, page, nodes
        self.max_context = context + room
        pages = -(-(self.max_context + nodes) // page)
        self.embed = rand(vocab, hidden).bfloat16()
        self.w_qkv = (rand((q_heads + 2 * kv_heads) * dim, hidden) * hidden**-0.5).bfloat16()
        self.w_o = (rand(hidden, q_heads * dim) * (q_heads * dim) ** -0.5).bfloat16()
        self.head = torch.randint(-127, 128, (vocab, hidden), generator=g, device=device, dtype=torch.int8)
        self.head_scale = (rand(vocab).abs() * (0.03 / 127)).bfloat16()
        self.table = fx.rotary_table(self.max_context + nodes, rotated, 1e6, fx.RotaryScaling(4.0), device=device)
        self.k_cache = rand(pages, page, kv_heads, dim).bfloat16()
        self.v_cache = rand(pages, page, kv_heads, dim).bfloat16()
        self.page_table = torch.randperm(pages, generator=g, device=device).to(torch.int32)[None]
        # what changes from step to step
        i32 = dict(dtype=torch.int32, device=device)
        self.context = torch.tensor([context], **i32)
        self.offsets = torch.tensor([0, nodes], **i32)
        self.parents = torch.full((nodes,), -1, **i32)
        self.tokens = torch.zeros(nodes, dtype=torch.int64, device=device)
        self.uniforms = torch.zeros(nodes, device=device)
        self.temperature = torch.full((nodes,), temperature, device=device)
        self.top_k = torch.full((nodes,), top_k, **i32)
        self.top_p = torch.full((nodes,), top_p, device=device)
        fx.prealloc(device, attention=True)

    def run(self):
        mask, positions, self.slots = fx.tree_layout(self.parents, self.offsets, self.context, self.page_table,
                                                     self.page, self.k_cache.shape[0])
        qkv = torch.cat([fx.bf16_gemv(x, self.w_qkv) for x in self.embed[self.tokens].split(16)])
        q, k, v = (x.unflatten(1, (-1, self.dim)) for x in qkv.split(
            [self.q_heads * self.dim, self.kv_heads * self.dim, self.kv_heads * self.dim], 1))
        q = fx.rotary_append(q, k, v, positions, self.slots, self.table, self.k_cache, self.v_cache)
        out, _ = fx.tree_attention(q, self.k_cache, self.v_cache, self.page_table, self.context, self.offsets, mask,
                                   max_nodes=self.nodes, max_context=self.max_context)
        hidden = torch.cat([fx.bf16_gemv(x, self.w_o) for x in out.flatten(1).split(16)])
        self.logits = torch.cat([fx.w8a16_gemv(x, self.head, self.head_scale) for x in hidden.split(16)])
        self.sampled, self.probs = fx.sample_tokens(self.logits, self.uniforms, self.temperature, self.top_k,
                                                    self.top_p)

    def accept(self):
        """([accepted drafted tokens], the token sampled after them); the context grows by node 0 and them."""
        parents, tokens, sampled = self.parents.tolist(), self.tokens.tolist(), self.sampled.tolist()
        path = [0]
        while True:
            child = next((j for j in range(path[-1] + 1, self.nodes)
                          if parents[j] == path[-1] and tokens[j] == sampled[path[-1]]), None)
            if child is None:
                break
            path.append(child)
        old, new = self.slots[path], self.slots[: len(path)]
        for cache in (self.k_cache, self.v_cache):
            rows = cache.view(-1, self.kv_heads, self.dim)
            rows[new] = rows[old]
        self.context += len(path)
        return [tokens[j] for j in path[1:]], sampled[path[-1]]

    def draft(self, last: int, generator: torch.Generator):
        """A random tree behind the token `last`; half of it guesses what will be sampled.  (A drafter's
        place: here the guesses come from a run over the tree itself.)"""
        cpu = torch.Generator().manual_seed(int(torch.randint(0, 2**31, (1,), generator=generator)))
        parents = [-1] + [int(torch.randint(max(0, i - 3), i, (1,), generator=cpu)) for i in range(1, self.nodes)]
        tokens = torch.randint(0, self.embed.shape[0], (self.nodes,), generator=cpu)
        tokens[0] = last
        self.parents.copy_(torch.tensor(parents, dtype=torch.int32))
        self.tokens.copy_(tokens)
        self.uniforms.copy_(torch.rand(self.nodes, generator=cpu))
        return parents


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--context", type=int, default=4000)
    ap.add_argument("--nodes", type=int, default=8)
    args = ap.parse_args(argv)
    step = VerifyStep(args.context, args.nodes)
    step.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run()
    generator = torch.Generator().manual_seed(1)
    last, text = 7, []
    for _ in range(args.steps):
        parents = step.draft(last, generator)
        graph.replay()
        # let some drafted tokens be right: a node that guesses what its parent's row samples
        for j in range(1, args.nodes, 2):
            step.tokens[j] = step.sampled[parents[j]]
            graph.replay()
        accepted, last = step.accept()
        text += accepted + [last]
        print(f"accepted {len(accepted)} of {args.nodes - 1} drafted tokens, context {int(step.context)}")
    fx.check_device_errors()
    print("tokens:", text)
    return text


if __name__ == "__main__":
    main()
