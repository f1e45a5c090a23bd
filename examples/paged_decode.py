"""A small decoder served from a paged key-value cache.

Random weights, a few layers. Prompts of different lengths are packed and prefilled (their keys and
values go to pages as the attention over the prompt runs); then every step appends one token for each
sequence, and attends over all of its pages or, with --budget, over the pages that score highest.

    python examples/paged_decode.py                       # all pages
    python examples/paged_decode.py --cache fp8 --budget 8
    python examples/paged_decode.py --check               # against recomputing every prefix
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from bytes_b200 import paged  # noqa: E402


class Decoder:
    """Attention blocks with a rotary embedding, RMS norms and a gated MLP, in bf16."""

    def __init__(self, layers=2, hidden=512, q_heads=8, kv_heads=2, head_dim=64, vocab=512, positions=4096, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*shape):
            return (torch.randn(shape, generator=g, device="cuda") * shape[-1] ** -0.5).bfloat16()

        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.embed, self.head = weight(vocab, hidden) * hidden ** 0.5, weight(vocab, hidden)
        self.layers = [dict(qkv=weight((q_heads + 2 * kv_heads) * head_dim, hidden), out=weight(hidden, q_heads * head_dim),
                            up=weight(4 * hidden, hidden), down=weight(hidden, 2 * hidden)) for _ in range(layers)]
        angle = torch.arange(positions, device="cuda").double()[:, None] * 10000.0 ** (
            -torch.arange(0, head_dim, 2, device="cuda").double() / head_dim)
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    def norm(self, x):
        return (x.float() * x.float().square().mean(-1, keepdim=True).add(1e-6).rsqrt()).bfloat16()

    def forward(self, tokens, attend):
        """tokens [T]; attend(layer number, q, k, v) -> [T, q_heads, head_dim]. Returns logits [T, vocab]."""
        x = self.embed[tokens]
        for i, w in enumerate(self.layers):
            qkv = (self.norm(x) @ w["qkv"].T).unflatten(1, (-1, self.head_dim))
            q, k, v = qkv.split([self.q_heads, self.kv_heads, self.kv_heads], 1)
            x = x + attend(i, q, k, v).flatten(1) @ w["out"].T
            a, b = (self.norm(x) @ w["up"].T).chunk(2, -1)
            x = x + (torch.nn.functional.silu(a) * b) @ w["down"].T
        return self.norm(x) @ self.head.T


class PagedCache:
    """Pages for every layer, one block table for all; pages are handed out from a free list."""

    def __init__(self, model, sequences, pages, block=16, dtype=torch.bfloat16, widest=256):
        shape = (pages, model.kv_heads, block, model.head_dim)
        self.k = [torch.zeros(shape, device="cuda", dtype=dtype) for _ in model.layers]
        self.v = [torch.zeros(shape, device="cuda", dtype=dtype) for _ in model.layers]
        self.summary = [paged.new_block_summary(k) for k in self.k]
        self.block, self.free = block, torch.randperm(pages).tolist()
        self.table = torch.full((sequences, widest), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(sequences, dtype=torch.int32, device="cuda")
        self.host_lens = [0] * sequences
        # what an 8-bit cache is scaled by; real models take theirs from data
        self.scales = dict(k_scale=0.05, v_scale=0.05) if dtype == torch.float8_e4m3fn else {}

    def grow(self, new):
        """Makes room for new[b] further tokens of sequence b, which then count as its length."""
        for b, n in enumerate(new):
            for j in range(-(-self.host_lens[b] // self.block), -(-(self.host_lens[b] + n) // self.block)):
                self.table[b, j] = self.free.pop()
            self.host_lens[b] += n
        self.lens += torch.tensor(new, dtype=torch.int32, device="cuda")


def prefill(model, cache, prompts):
    """All prompts in one packed pass; logits of each prompt's last token."""
    new = [p.numel() for p in prompts]
    cu = torch.tensor([0] + new).cumsum(0)
    cache.grow(new)
    dev_cu = cu.int().cuda()

    def attend(i, q, k, v):
        # pages take the rotated keys; the prompt's own attention reads them back from the same call's output
        code, scale = cache.summary[i]
        q = paged.paged_append(k, v, cache.k[i], cache.v[i], cache.table, cache.lens, q=q, cos=model.cos, sin=model.sin,
                               cu_seqlens=dev_cu, summary=code, summary_scale=scale, **cache.scales)
        out = torch.empty_like(q)
        for b, n in enumerate(new):
            at = cache.table[b, :-(-n // cache.block)].long()
            kb, vb = (c[i][at].transpose(1, 2).flatten(0, 1)[:n].float() for c in (cache.k, cache.v))
            kb, vb = kb * cache.scales.get("k_scale", 1.0), vb * cache.scales.get("v_scale", 1.0)
            rows = slice(int(cu[b]), int(cu[b + 1]))
            out[rows] = torch.nn.functional.scaled_dot_product_attention(
                q[rows].transpose(0, 1).float()[None], kb.transpose(0, 1)[None], vb.transpose(0, 1)[None], is_causal=True,
                enable_gqa=True)[0].transpose(0, 1).to(out.dtype)
        return out

    return model.forward(torch.cat(prompts), attend)[cu[1:].cuda() - 1]


def step(model, cache, tokens, budget=0):
    """One new token for each sequence; its logits."""
    cache.grow([1] * tokens.numel())
    scaling = model.head_dim ** -0.5

    def attend(i, q, k, v):
        code, scale = cache.summary[i]
        q = paged.paged_append(k, v, cache.k[i], cache.v[i], cache.table, cache.lens, q=q, cos=model.cos, sin=model.sin,
                               summary=code, summary_scale=scale, **cache.scales)
        if budget:
            return paged.paged_sparse_decode_attn(q, cache.k[i], cache.v[i], code, scale, cache.table, cache.lens, budget,
                                                  scaling, sink_blocks=1, recent_blocks=2, **cache.scales)
        return paged.paged_decode_attn(q, cache.k[i], cache.v[i], cache.table, cache.lens, scaling, **cache.scales)

    return model.forward(tokens, attend)


def recompute(model, tokens):
    """Logits of the last of `tokens` without a cache."""
    n = tokens.numel()

    def attend(i, q, k, v):
        def turn(x):
            a, b = x.float().chunk(2, -1)
            c, s = model.cos[:n, None], model.sin[:n, None]
            return torch.cat([a * c - b * s, b * c + a * s], -1).bfloat16().float()
        q, k, v = (x.transpose(0, 1)[None].float() for x in (turn(q), turn(k), v))
        return torch.nn.functional.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)[0] \
            .transpose(0, 1).bfloat16()

    return model.forward(tokens, attend)[-1]


def generate(prompt_lens, steps, dtype=torch.bfloat16, budget=0, seed=0):
    """(model, prompts, forced tokens [steps, B], logits [steps + 1, B, vocab]): tokens are drawn, not the
    logits' own, so that runs can be compared step by step."""
    model = Decoder(seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    prompts = [torch.randint(0, 512, (n,), generator=g, device="cuda") for n in prompt_lens]
    forced = torch.randint(0, 512, (steps, len(prompts)), generator=g, device="cuda")
    pages = sum(-(-(n + steps) // 16) for n in prompt_lens) + 1
    cache = PagedCache(model, len(prompts), pages, dtype=dtype)
    logits = [prefill(model, cache, prompts)]
    for t in range(steps):
        logits.append(step(model, cache, forced[t], budget))
    return model, prompts, forced, torch.stack(logits)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--cache", choices=("bf16", "fp8"), default="bf16")
    ap.add_argument("--budget", type=int, default=0, help="pages that a step attends over (0: all)")
    ap.add_argument("--steps", type=int, default=24)
    ap.add_argument("--check", action="store_true", help="compare every step with recomputing its prefix")
    a = ap.parse_args()
    dtype = torch.float8_e4m3fn if a.cache == "fp8" else torch.bfloat16
    model, prompts, forced, logits = generate([5, 130, 333, 1000], a.steps, dtype, a.budget)
    print("logits", tuple(logits.shape), "greedy tokens of the last step:", logits[-1].argmax(-1).tolist())
    if a.check:
        worst = 0.0
        for b, p in enumerate(prompts):
            for t in range(a.steps + 1):
                want = recompute(model, torch.cat([p, forced[:t, b]])).float()
                worst = max(worst, float((logits[t, b].float() - want).norm() / want.norm()))
        print("largest relative difference from recomputing: %.3g" % worst)


if __name__ == "__main__":
    main()
