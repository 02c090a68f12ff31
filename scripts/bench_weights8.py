#!/usr/bin/env python
"""Whole models with their Linears in 16 and in 8 bits (Transformer.quantise_weights), the same loops on the same GPU: prompts with the logits of all their rows, and decode steps behind a
context, on rings and on pages.  Random weights.  Usage: python scripts/bench_weights8.py [--head] [model ...]      (--head: the lm head in 8 bits too)

Prompts: the median of 7 timed calls behind 2 others, a fresh cache each.  Steps: 64 behind 32 others, each fed the step before's own pick.  Every step and prompt reads the
model's weights, more than L2 holds.  And the rotation and cache phase behind the query, key and value product by itself, over inputs of some 300 MB in turn."""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import synth  # noqa: E402
import mistral_inference_b200 as mi  # noqa: E402
from mistral_inference_b200 import _abi_rows8  # noqa: E402

PROMPTS = (128, 777, 2048, 4096)
STEPS = {"mistral-7b": (1, 4000), "mistral-nemo-12b": (32, 1024)}  # sequences, tokens ahead of the first step


def model_of(name, batch):
    p = synth.shape(name)
    args = mi.TransformerArgs.from_dict(dict(p))
    args.max_batch_size = batch
    m = mi.Transformer.empty(args, "cuda", torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(1)
    for w in m.parameters():
        w.data.normal_(0.0, w.shape[-1] ** -0.5, generator=g) if w.dim() > 1 else w.data.fill_(1.0)
    return m.eval(), p


def milliseconds(f):
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    a.record()
    f()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b)


def prompt(m, p, tokens):
    ids = torch.randint(0, p["vocab_size"], (tokens,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(tokens))
    times = []
    for _ in range(9):
        cache = m.make_cache(1, tokens + 8)
        times.append(milliseconds(lambda: m.forward(ids, [tokens], cache)))
    return sorted(times[2:])[3]


def step(m, p, batch, past, kv_cache):
    cache = m.make_cache(batch, past + 128, kv_cache=kv_cache)
    ids = torch.randint(0, p["vocab_size"], (batch * past,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(past))
    _, logits = m.forward_logprobs(ids, [past] * batch, cache, torch.full_like(ids, -1))
    tok = logits.argmax(-1)

    def steps(n):
        nonlocal tok
        for _ in range(n):
            m.decode_static(tok, cache)
            tok = m.last_argmax
    steps(32)
    return milliseconds(lambda: steps(64)) / 64


def rotation(tokens, heads, kv):
    copies = max(2, (300 << 20) // (tokens * (heads + 2 * kv) * 512) + 1)
    copies = min(copies, 256)
    qkv = [torch.randn(tokens, (heads + 2 * kv) * 128, device="cuda").bfloat16() for _ in range(copies)]
    outs = [[torch.empty(tokens, n * 128, device="cuda", dtype=torch.bfloat16) for n in (heads, kv, kv)] for _ in range(copies)]
    rope, positions = torch.randn(8192, 64, 2, device="cuda"), torch.arange(tokens, device="cuda", dtype=torch.int32)

    def run():
        for x, o in zip(qkv, outs):
            _abi_rows8.rotate(x, rope, positions, None, *o, heads, kv)
    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    g.replay()
    us = milliseconds(lambda: [g.replay() for _ in range(8)]) / 8 / copies * 1e3
    return us, tokens * (heads + 2 * kv) * 512 / us / 1e3


def main():
    names = [a for a in sys.argv[1:] if a != "--head"] or list(STEPS)
    for name in names:
        batch, past = STEPS[name]
        m, p = model_of(name, batch)
        got = []
        for weights in ("16 bits", "8 bits"):
            if weights == "8 bits":
                m.quantise_weights(head="--head" in sys.argv)
            row = [("prompt %d" % t, prompt(m, p, t)) for t in PROMPTS] if batch == 1 else []
            row += [("step %d x %d, %s" % (batch, past, kv), step(m, p, batch, past, kv)) for kv in ("ring", "pages")]
            got.append(row)
        for (what, a), (_, b) in zip(*got):
            print(f"{name:18s} {what:24s} ms: 16 bits {a:8.3f}   8 bits {b:8.3f}", flush=True)
        del m
        torch.cuda.empty_cache()
    for tokens in (1, 32, 777, 4096):
        us, gbs = rotation(tokens, 32, 8)
        print(f"rotation of {tokens:5d} tokens, 32 + 2 * 8 heads: {us:7.2f} us, {gbs:7.1f} GB/s", flush=True)


if __name__ == "__main__":
    main()
