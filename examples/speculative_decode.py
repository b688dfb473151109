#!/usr/bin/env python3
"""Drafted decoding of a small decoder on the serving operators.

    python examples/speculative_decode.py [--new 48] [--dtype bf16]

A two-layer decoder with random weights, grouped heads and rotary positions
answers a packed batch of prompts:

* prompts     rope_append (rotated queries; rotated keys and values into the
              pages), prompt_attention
* each step   a tree of tokens guessed from the pairs seen so far, its mask
              from tree_mask; rope_append, tree_attention; the longest branch
              that the model itself would have taken is kept, cache_accept
              moves its cache entries up in every layer

The projections are the framework's fp16 GEMMs (kbt_sgemm, and
kbt_gemm_rmsnorm_swiglu for the gated half of the feed-forward), so with
dtype f16 the whole step runs on its kernels; bf16 uses torch's products.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from akili_bench_b200 import ops  # noqa: E402

VOCAB, DIM, LAYERS, Q_HEADS, KV_HEADS, HEAD_DIM, FFN = 256, 256, 2, 8, 2, 64, 512
PAGE, MAX_POSITIONS = 16, 1024


def weights(dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = lambda *s: (torch.randn(s, generator=g, device="cuda") * s[0] ** -0.5).to(dtype)  # noqa: E731
    layers = [{"qkv": w(DIM, (Q_HEADS + 2 * KV_HEADS) * HEAD_DIM), "o": w(Q_HEADS * HEAD_DIM, DIM),
               "gate": w(DIM, FFN), "up": w(DIM, FFN), "down": w(FFN, DIM)} for _ in range(LAYERS)]
    embed = torch.randn(VOCAB, DIM, generator=g, device="cuda").to(dtype)
    return {"embed": embed, "layers": layers, "head": (w(DIM, VOCAB).float() * 2).to(dtype)}


def product(x, w):
    """x.w; fp16 on the framework's GEMM, whose rows come in eights."""
    if x.dtype != torch.float16:
        return x @ w
    pad = -x.shape[0] % 8
    return ops.kbt_sgemm(torch.nn.functional.pad(x, (0, 0, 0, pad)), w, out_dtype=torch.float16)[:x.shape[0]]


def gated(x, gate, up):
    """silu(norm(x).gate) * (norm(x).up)."""
    if x.dtype != torch.float16:
        y = norm(x)
        return torch.nn.functional.silu((y @ gate).float()).mul((y @ up).float()).to(x.dtype)
    pad = -x.shape[0] % 8
    ones = torch.ones(DIM, device=x.device)
    return ops.kbt_gemm_rmsnorm_swiglu(torch.nn.functional.pad(x, (0, 0, 0, pad)), ones, gate, up)[:x.shape[0]]


def norm(x):
    y = x.float()
    return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5)).to(x.dtype)


class Decoder:
    def __init__(self, dtype, batch, capacity):
        self.w = weights(dtype)
        self.table = ops.rope_table(MAX_POSITIONS, HEAD_DIM)
        per = -(-capacity // PAGE)
        shape = (LAYERS, batch * per, PAGE, KV_HEADS, HEAD_DIM)
        self.k_pages, self.v_pages = (torch.empty(shape, dtype=dtype, device="cuda") for _ in range(2))
        self.page_table = torch.randperm(batch * per, device="cuda").to(torch.int32).view(batch, per)
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def forward(self, tokens, sequence, entry, positions, cu, mask=None, prompt=False):
        """Logits of packed tokens; `entry` is each one's place in its sequence's cache."""
        slots = self.page_table[sequence, entry // PAGE].long() * PAGE + entry % PAGE
        positions = positions.to(torch.int32)
        x = self.w["embed"][tokens]
        for i, layer in enumerate(self.w["layers"]):
            qkv = product(norm(x), layer["qkv"]).view(-1, Q_HEADS + 2 * KV_HEADS, HEAD_DIM)
            q, k, v = qkv.split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
            pages = self.k_pages[i], self.v_pages[i]
            q = ops.rope_append(q, k, v, positions, self.table, slots, *pages, k_out=k if prompt else None)
            if prompt:
                o = ops.prompt_attention(q, k, v, cu)
            else:
                o = ops.tree_attention(q, *pages, self.page_table, self.lens, cu, mask)
            x = x + product(o.flatten(1), layer["o"])
            x = x + product(gated(x, layer["gate"], layer["up"]), layer["down"])
        return product(norm(x), self.w["head"])

    def prompts(self, prompts):
        """Fills the cache; the first new token of each sequence."""
        lens = torch.tensor([len(p) for p in prompts])
        cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)])
        sequence = torch.arange(len(prompts)).repeat_interleave(lens)
        at = (torch.arange(int(cu[-1])) - cu[sequence]).cuda()
        logits = self.forward(torch.tensor(sum(prompts, []), device="cuda"), sequence.cuda(), at, at,
                              cu.to(torch.int32).cuda(), prompt=True)
        self.lens = lens.to(torch.int32).cuda()
        return logits[(cu[1:] - 1).cuda()].argmax(-1).tolist()

    def step(self, trees):
        """Verifies one tree per sequence ([(token, parent)], node 0 the newest sure token); the tokens it yields."""
        nodes = [len(t) for t in trees]
        start = [sum(nodes[:b]) for b in range(len(nodes) + 1)]
        cu = torch.tensor(start, dtype=torch.int32, device="cuda")
        depth = []
        for t in trees:
            d = []
            for _, parent in t:
                d.append(0 if parent < 0 else d[parent] + 1)
            depth += d
        dev = lambda v, dt=torch.long: torch.tensor(v, dtype=dt, device="cuda")  # noqa: E731
        parents = dev([p for t in trees for _, p in t], torch.int32)
        sequence = dev([b for b, n in enumerate(nodes) for _ in range(n)])
        index = dev([i for n in nodes for i in range(n)])
        base = self.lens[sequence]
        mask = ops.tree_mask(parents, cu, max(nodes))
        logits = self.forward(dev([x for t in trees for x, _ in t]), sequence, base + index, base + dev(depth), cu, mask)
        best = logits.argmax(-1).tolist()
        kept, yielded = [], []
        for b, t in enumerate(trees):
            node, path, out = 0, [0], [best[start[b]]]
            while True:  # the child that the model chose, if it was drafted
                child = [i for i, (x, p) in enumerate(t) if p == node and x == out[-1]]
                if not child:
                    break
                node = child[0]
                path.append(node)
                out.append(best[start[b] + node])
            kept.append(path)
            yielded.append(out)
        most = max(len(p) for p in kept)
        self.lens = ops.cache_accept(self.k_pages, self.v_pages, self.page_table, self.lens,
                                     dev([p + [0] * (most - len(p)) for p in kept], torch.int32),
                                     dev([len(p) for p in kept], torch.int32))
        return yielded


def draft(tokens, width=2, depth=4, most=12):
    """A tree after the last token: what followed each token before, latest first."""
    after = {}
    for a, b in zip(tokens, tokens[1:]):
        after.setdefault(a, []).insert(0, b)
    tree = [(tokens[-1], -1)]
    level = [0]
    for _ in range(depth):
        grown = []
        for node in level:
            for x in list(dict.fromkeys(after.get(tree[node][0], [])))[:width]:
                if len(tree) < most:
                    grown.append(len(tree))
                    tree.append((x, node))
        level = grown
    return tree


def generate(prompts, new, dtype, drafted=True):
    """(tokens of each sequence, steps taken)."""
    room = max(len(p) for p in prompts) + new + 32
    model = Decoder(dtype, len(prompts), room)
    seqs = [list(p) for p in prompts]
    for s, x in zip(seqs, model.prompts(prompts)):
        s.append(x)
    steps = 0
    while min(len(s) - len(p) for s, p in zip(seqs, prompts)) < new:
        trees = [draft(s) if drafted and len(s) - len(p) < new else [(s[-1], -1)] for s, p in zip(seqs, prompts)]
        for s, p, out in zip(seqs, prompts, model.step(trees)):
            if len(s) - len(p) < new:
                s += out
        steps += 1
        # the cache holds all but the newest token (a finished sequence repeats its last step)
        model.lens = torch.tensor([len(s) - 1 for s in seqs], dtype=torch.int32, device="cuda")
    return [s[:len(p) + new] for s, p in zip(seqs, prompts)], steps


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--new", type=int, default=48)
    ap.add_argument("--dtype", choices=("f16", "bf16"), default="f16")
    a = ap.parse_args()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in (37, 5, 150)]
    dtype = torch.float16 if a.dtype == "f16" else torch.bfloat16
    seqs, steps = generate(prompts, a.new, dtype)
    _, plain = generate(prompts, a.new, dtype, drafted=False)
    for p, s in zip(prompts, seqs):
        print(f"prompt of {len(p):3d}: {s[len(p):]}")
    print(f"{a.new} tokens each in {steps} steps ({plain} without drafts); device status {ops.device_status()}")


if __name__ == "__main__":
    main()
