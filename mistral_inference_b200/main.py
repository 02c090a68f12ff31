"""Command line: `python -m mistral_inference_b200.main generate MODEL_DIR --prompt "5 17 3" [--prompt ...] --max-tokens N`.

Loads any model folder through the registry (reference-format `params.json` checkpoints and `config.json` designs alike) and
runs `generate()` on prompts given as token ids (no tokenizer ships with these checkpoints; the reference's `mistral-demo`,
main.py:163-196, does the same job after tokenising).  Prints one line of generated ids per prompt (and one per token with --alternatives).
"""
import argparse
import sys
from typing import List, Optional


def main(argv: Optional[List[str]] = None) -> int:
    ap = argparse.ArgumentParser(prog="mistral_inference_b200")
    sub = ap.add_subparsers(dest="cmd", required=True)
    g = sub.add_parser("generate", help="greedy or nucleus generation from prompts of token ids")
    g.add_argument("model")
    g.add_argument("--prompt", action="append", required=True, help="token ids separated by spaces; repeat for a batch")
    g.add_argument("--max-tokens", type=int, default=32)
    g.add_argument("--temperature", type=float, default=0.0)
    g.add_argument("--chunk-size", type=int, default=None)
    g.add_argument("--dtype", choices=["bfloat16", "float32"], default=None)
    g.add_argument("--kv-cache", choices=["ring", "pages"], default="ring", help="keys and values in 16-bit rings, or in 8-bit pages (reference-format checkpoints)")
    g.add_argument("--alternatives", type=int, default=0, help="print that many of the most likely tokens at every generated one, with its log-probability and entropy")
    a = ap.parse_args(argv)

    import torch

    from .generate import generate
    from .registry import load_model

    prompts = [[int(t) for t in p.split()] for p in a.prompt]
    model = load_model(a.model, max_batch_size=len(prompts), dtype=getattr(torch, a.dtype) if a.dtype else None)
    out = generate(prompts, model, max_tokens=a.max_tokens, temperature=a.temperature, chunk_size=a.chunk_size, kv_cache=a.kv_cache, alternatives=a.alternatives)
    for b, row in enumerate(out[0]):
        print(" ".join(str(t) for t in row))
        if a.alternatives:
            for t, lp, d in zip(row, out[1][b][len(prompts[b]) - 1:], out[2][b][len(prompts[b]) - 1:]):
                print(f"  {t}  logprob {lp:.4f}  entropy {d.entropy:.4f}  " + " ".join(f"{i}:{p:.4f}" for i, p in zip(d.top_ids, d.top_logprobs)))
    return 0


if __name__ == "__main__":
    sys.exit(main())
