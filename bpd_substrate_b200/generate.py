"""Command line: generation from token ids, greedy or sampled.

    python -m bpd_substrate_b200.generate --model DIR_OR_GGUF --prompt "5 17 3" [--prompt ...] --max-new 32 [--temperature 0.8 --top-k 40 --top-p 0.95 --min-p 0.05 --seed 1]
"""
import argparse
import json
import sys

from .engine import Engine
from .registry import load_model
from .sampling import Sampling


def main(argv=None):
    ap = argparse.ArgumentParser(prog="generate", description="Generation from token ids; one JSON line per prompt.")
    ap.add_argument("--model", required=True, help="model folder (config.json, model.safetensors) or .gguf file")
    ap.add_argument("--prompt", action="append", required=True, help="token ids, separated by blanks or commas; may be repeated")
    ap.add_argument("--max-new", type=int, default=16)
    ap.add_argument("--stop", type=int, action="append", default=[], help="token id that ends a generation; may be repeated")
    ap.add_argument("--dtype", choices=("bfloat16", "float32"), default="bfloat16")
    ap.add_argument("--capacity", type=int, default=4096, help="tokens a sequence may hold")
    ap.add_argument("--slots", type=int, default=4, help="sequences in memory at once")
    ap.add_argument("--portion", type=int, default=2048, help="most prompt tokens per step")
    ap.add_argument("--temperature", type=float, default=0.0, help="0: greedy")
    ap.add_argument("--top-k", type=int, default=0, help="only the k likeliest tokens; 0: all")
    ap.add_argument("--top-p", type=float, default=1.0, help="only the likeliest tokens that have this share between them")
    ap.add_argument("--min-p", type=float, default=0.0, help="only tokens at least this likely, of the likeliest one")
    ap.add_argument("--seed", type=int, default=0, help="of the random numbers; the next prompt takes the next one")
    a = ap.parse_args(argv)
    sampling = Sampling(a.temperature, a.top_k, a.top_p, a.min_p, a.seed) if a.temperature else None
    prompts = [[int(t) for t in p.replace(",", " ").split()] for p in a.prompt]
    model = load_model(a.model, a.dtype, a.capacity)
    engine = Engine(model, min(a.slots, len(prompts)), a.portion)
    try:
        for p, out in zip(prompts, engine.generate(prompts, a.max_new, a.stop, sampling)):
            print(json.dumps({"prompt": p, "output": out}), flush=True)
    finally:
        engine.close()
        model.close()
    return 0


if __name__ == "__main__":
    sys.exit(main())
