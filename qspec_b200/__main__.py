"""Command line of the framework.

    python -m qspec_b200 models                                   architectures the registry knows
    python -m qspec_b200 generate --model DIR --prompt 5,17,3 [--prompt ...] [--max-new-tokens N] [--dtype bfloat16]
    python -m qspec_b200 score --model DIR --prompt 5,17,3 [--prompt ...] [--top N] [--dtype bfloat16]
    python -m qspec_b200 trace --model DIR --dtype ... --out DIR  replay recorded steps (qspec_b200/trace.py)
    python -m qspec_b200 build [--seq]                            compile the kernel libraries

`generate` takes prompts as comma-separated token ids (the framework has no tokenizer), runs them through the
continuous-batching scheduler with greedy sampling and prints one JSON line per prompt (with --logprobs N also each token's log probability, rank, entropy and N
alternatives). `score` prints the same of given tokens, and the text's perplexity. Numbers that are infinite, or none, are null.
"""
from __future__ import annotations

import argparse
import json
import math
import sys
from dataclasses import asdict


def _arguments(command: str) -> argparse.ArgumentParser:
    ap = argparse.ArgumentParser(prog=f"python -m qspec_b200 {command}")
    ap.add_argument("--model", required=True, help="folder with config.json (and weights)")
    ap.add_argument("--dtype", default=None, help="bfloat16 | float32 | float16 (default: the model's serving type)")
    ap.add_argument("--prompt", action="append", required=True, help="comma-separated token ids; repeat for several prompts")
    ap.add_argument("--slots", type=int, default=8)
    ap.add_argument("--step-tokens", type=int, default=2048)
    ap.add_argument("--prefill-portion", type=int, default=None, help="most prompt tokens of one request per step")
    ap.add_argument("--kv-cache", default=None, choices=("f16", "int8", "uint4"), help="of the int4 decoders: rows of 16 bits, or pages of 8-bit or 4-bit codes")
    return ap


def _scheduler(args, new_tokens: int):
    """The scheduler over the model that the arguments name, and the prompts."""
    from . import registry
    from .build import build_library, build_seq_library
    arch = registry.architecture_of(registry.read_config(args.model))
    if args.kv_cache and arch in registry.SEQUENCE_DESIGNS:
        raise SystemExit(f"--kv-cache is for the int4 decoders, not {arch}")
    build_seq_library()
    if arch not in registry.SEQUENCE_DESIGNS:
        build_library()
    from .scheduler import Scheduler
    prompts = [[int(t) for t in p.split(",") if t.strip()] for p in args.prompt]
    # models whose cache grows with the sequence size it for the longest request
    model = registry.load_model(args.model, dtype=args.dtype, n_slots=args.slots, max_step_tokens=args.step_tokens,
                                max_seq_tokens=max(len(p) for p in prompts) + new_tokens, **({"kv_cache": args.kv_cache} if args.kv_cache else {}))
    return Scheduler(model, prefill_portion=args.prefill_portion), prompts


def _print(line: dict) -> None:
    def plain(x):
        if isinstance(x, dict):
            return {k: plain(v) for k, v in x.items()}
        if isinstance(x, (list, tuple)):
            return [plain(v) for v in x]
        return None if isinstance(x, float) and not math.isfinite(x) else x
    print(json.dumps(plain(line), allow_nan=False))


def _generate(argv) -> int:
    ap = _arguments("generate")
    ap.add_argument("--max-new-tokens", type=int, default=16)
    ap.add_argument("--eos", type=int, default=None)
    ap.add_argument("--logprobs", type=int, default=None, help="log probabilities of the tokens, with so many alternatives")
    args = ap.parse_args(argv)
    scheduler, prompts = _scheduler(args, args.max_new_tokens)
    for p, r in zip(prompts, scheduler.generate_requests(prompts, args.max_new_tokens, args.eos, args.logprobs)):
        _print({"prompt": p, "tokens": r.output} | ({} if args.logprobs is None else {"scores": [asdict(s) for s in r.scores]}))
    return 0


def _score(argv) -> int:
    ap = _arguments("score")
    ap.add_argument("--top", type=int, default=0, help="alternatives of each place")
    args = ap.parse_args(argv)
    scheduler, prompts = _scheduler(args, 0)
    for p, scores in zip(prompts, scheduler.score(prompts, args.top)):
        mean = sum(s.logprob for s in scores) / len(scores) if scores else math.nan
        _print({"prompt": p, "perplexity": math.exp(-mean) if mean > -700 else None, "scores": [asdict(s) for s in scores]})
    return 0


def main(argv=None) -> int:
    argv = list(sys.argv[1:] if argv is None else argv)
    if not argv or argv[0] in ("-h", "--help"):
        print(__doc__)
        return 0
    cmd, rest = argv[0], argv[1:]
    if cmd == "models":
        from . import registry
        print("\n".join(registry.architectures()))
        return 0
    if cmd == "generate":
        return _generate(rest)
    if cmd == "score":
        return _score(rest)
    if cmd == "trace":
        from .trace import main as trace_main
        return trace_main(rest)
    if cmd == "build":
        from .build import build_library, build_seq_library
        print(build_seq_library(force="--force" in rest, verbose=True) if "--seq" in rest
              else build_library(force="--force" in rest, verbose=True))
        return 0
    print(f"unknown command {cmd!r}\n{__doc__}", file=sys.stderr)
    return 2


if __name__ == "__main__":
    sys.exit(main())
