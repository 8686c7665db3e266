#!/usr/bin/env python3
"""Answers questions over the passages that a search finds, on one GPU.

A small transformer with random weights (layers of attention alone, no
training) stands in for a model; what matters is the order of the calls:

1. Passages of different lengths go through the model in one packed batch,
   each token seeing its whole passage (prompt attention, not causal); the mean
   of a passage's tokens is its vector, and the vectors become a dataset.
2. The topic that the questions share is searched for: exact k-NN.
3. The passages found go through the model once, one behind another, as the
   beginning of a prompt (prompt attention, causal), and their keys and values
   into a paged cache.
4. Every question's sequence forks that cache, is extended by its own tokens,
   which attend to the passages and themselves, and then generates token by
   token, all questions of the batch together: the passages' pages are read
   once a step for all of them.
5. Half of the sequences end and the cache is compacted; each answer is checked
   against the whole prompt run through prompt attention from scratch.

Positions are added to the tokens' embeddings, or (positions="rotary") turn
the queries and keys, whose heads are normed first: of a prompt in one pass
before its attention, of new tokens on their way into the cache.

Run: python examples/answer_over_passages.py [rotary]
"""
from __future__ import annotations

import importlib.util
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load_package():
    name = "cuvs_silicon_amd"
    if name not in sys.modules:
        pkg = os.path.join(ROOT, "cuvs-silicon_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


class Model:
    """Layers of grouped-head attention with residuals; random weights."""

    def __init__(self, seed, vocab=1000, width=512, layers=3, heads=8, kv_heads=2, dim=64, dtype=torch.float16,
                 added=True):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*shape):
            return (torch.randn(*shape, generator=g, device="cuda") / math.sqrt(shape[0])).to(dtype)

        self.layers, self.heads, self.kv_heads, self.dim, self.width = layers, heads, kv_heads, dim, width
        self.tokens = torch.randn(vocab, width, generator=g, device="cuda").to(dtype)
        self.qkv = [weight(width, (heads + 2 * kv_heads) * dim) for _ in range(layers)]
        self.out = [weight(heads * dim, width) for _ in range(layers)]
        half = torch.arange(width // 2, device="cuda") / (width // 2)
        self.frequencies = 1e-4 ** half
        self.added = added
        self.q_norm, self.k_norm = (torch.ones(dim, dtype=dtype, device="cuda") for _ in "qk")

    def embed(self, ids, positions):
        if not self.added:
            return self.tokens[ids]
        angle = positions[:, None].float() * self.frequencies
        return self.tokens[ids] + torch.cat([angle.sin(), angle.cos()], dim=1).to(self.tokens.dtype)

    def run(self, ids, positions, attend):
        """Hidden states of packed tokens; attend(layer, q, k, v, out) is the attention."""
        x = self.embed(ids, positions)
        for layer in range(self.layers):
            norm = x.float()
            norm = (norm * norm.square().mean(1, keepdim=True).add(1e-6).rsqrt()).to(x.dtype)
            qkv = (norm @ self.qkv[layer]).view(len(ids), self.heads + 2 * self.kv_heads, self.dim)
            q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
            out = torch.empty(len(ids), self.heads, self.dim, dtype=x.dtype, device="cuda")
            attend(layer, q, k, v, out)
            x = x + out.view(len(ids), -1) @ self.out[layer]
        return x

    def logits(self, x):
        return x.float() @ self.tokens.float().T


def packed_positions(lengths, first=0):
    return torch.cat([torch.arange(first, first + n, device="cuda") for n in lengths])


def main(passages=200, found=8, questions=12, steps=16, seed=1, quiet=False, positions="added"):
    say = (lambda *a: None) if quiet else print
    cvs = load_package()
    # A context on torch's stream: its calls and torch's run in order, and nothing is waited for in between.
    ctx = cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    model = Model(seed, added=positions == "added")
    rotary = ctx.rotary(model.dim) if positions == "rotary" else None

    def prompt(plan, places):
        """A prompt's attention: its queries and keys normed and turned in place, if the model has them so."""
        def attend(layer, q, k, v, out):
            if rotary:
                ctx.norm_rotate_async(rotary, places, q, q, k, k, model.q_norm, model.k_norm)
            ctx.prompt_attention_async(plan, q, k, v, out)
        return attend

    def run(ids, places, attend):
        return model.run(ids, places, attend(places))

    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(20, 200, (passages,), generator=g).tolist()
    texts = [torch.randint(1000, (n,), generator=g).cuda() for n in lengths]

    # 1. The passages' vectors.
    plan = ctx.prompt_plan(lengths, model.heads, model.kv_heads, causal=False)
    x = run(torch.cat(texts), packed_positions(lengths), lambda places: prompt(plan, places))
    owner = torch.repeat_interleave(torch.arange(passages, device="cuda"), torch.tensor(lengths, device="cuda"))
    vectors = torch.zeros(passages, model.width, device="cuda").index_add_(0, owner, x.float())
    vectors /= torch.tensor(lengths, device="cuda")[:, None]
    dataset = ctx.dataset(vectors.cpu().numpy())

    # 2. The passages nearest to a topic: here to the vector of one of them, with some noise.
    topic = vectors[7:8].cpu() + 0.01 * torch.randn(1, model.width, generator=g)
    ids, distances = dataset.bf_search(topic.numpy(), found)
    say("passages found:", ids[0].tolist())
    assert ids[0, 0] == 7

    # 3. The prompt's beginning, once, into the cache.
    prefix = torch.cat([texts[i] for i in ids[0]])
    page = 32
    asked = torch.randint(3, 40, (questions,), generator=g).tolist()
    pages = -(-len(prefix) // page) + sum(-(-(n + steps) // page) + 1 for n in asked)
    cache = ctx.kv_cache(model.layers, pages, page, model.kv_heads, model.dim, "fp16")
    root = cache.sequence()
    cache.extend([root], [len(prefix)])
    rows = cache.plan([root], [len(prefix)])
    plan = ctx.prompt_plan([len(prefix)], model.heads, model.kv_heads)

    def first_time(places):
        attend = prompt(plan, places)

        def and_keep(layer, q, k, v, out):
            attend(layer, q, k, v, out)
            cache.write_async(rows, k, v, layer=layer)
        return and_keep

    run(prefix, packed_positions([len(prefix)]), first_time)

    # 4. The questions, then their answers.
    own = [torch.randint(1000, (n,), generator=g).cuda() for n in asked]
    sequences = cache.fork(root, questions)
    new, last = list(asked), torch.cat(own)
    history, answer_logits = [t.clone() for t in own], []
    for step in range(steps):
        start = cache.lengths(sequences)
        cache.extend(sequences, new)
        rows = cache.plan(sequences, new, heads=model.heads)

        def over_cache(layer, q, k, v, out):
            if rotary:  # at the tokens' places in their sequences, which the plan knows
                cache.append_async(rows, k, v, layer=layer, rotary=rotary, k_weight=model.k_norm, q=q, q_out=q,
                                   q_weight=model.q_norm)
            else:
                cache.write_async(rows, k, v, layer=layer)
            cache.attention_async(rows, q, out, layer=layer)

        places = torch.cat([torch.arange(s, s + n, device="cuda") for s, n in zip(start, new)])
        x = run(last, places, lambda _: over_cache)
        ends = torch.tensor(new, device="cuda").cumsum(0) - 1
        answer_logits.append(model.logits(x[ends]))
        last = answer_logits[-1].argmax(1)
        history = [torch.cat([h, last[i:i + 1]]) for i, h in enumerate(history)]
        new = [1] * questions
    say(f"{questions} answers of {steps} tokens over {len(prefix)} shared tokens; "
        f"{cache.free_pages()} of {pages} pages free")

    # 5. Half of the sequences end; the others could go on from where compaction puts their pages.
    cache.free(sequences[::2] + [root])
    live = cache.compact()
    say(f"{live} pages live after compaction")
    worst = 0.0
    for i in range(questions):
        whole = torch.cat([prefix, history[i][:-1]])
        plan = ctx.prompt_plan([len(whole)], model.heads, model.kv_heads)
        x = run(whole, packed_positions([len(whole)]), lambda places: prompt(plan, places))
        want = model.logits(x[len(prefix) + asked[i] - 1:])
        got = torch.stack([l[i] for l in answer_logits])
        worst = max(worst, ((got - want).norm() / want.norm()).item())
    say(f"logits against the whole prompts from scratch: {worst:.2e} off (2-norm)")
    # Both routes round every layer's activations to fp16, at different places of the same sums.
    assert worst < 2e-2, worst
    cache.close()
    dataset.close()
    ctx.close()
    return worst


if __name__ == "__main__":
    main(positions="rotary" if "rotary" in sys.argv[1:] else "added")
