"""Answers prompts of token ids with a trained model (the reference trains only).

Example:  python generate.py --preset hybrid_1b --ckpt-root checkpoints --prompt 17,4,256 --prompt 9 \
              --max-new-tokens 64 --temperature 0.8 --top-p 0.95
Without ``--ckpt-root`` the weights are freshly initialised (for timing).  Prints one JSON line per
prompt: its tokens and their log-probabilities.  ``--prompt-file``: one prompt of comma-separated ids a line.
``--prefix``: ids that come before every prompt, read once for all.  ``--score N``: instead of answering, prints how likely
the model finds each prompt's own tokens, with the entropies and the N likeliest tokens at each place.
"""
import argparse
import json
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import torch  # noqa: E402

from atomic_ai_hybrid_b200.config import get_preset, load_yaml_config  # noqa: E402
from atomic_ai_hybrid_b200.models import HybridMoEModel  # noqa: E402
from atomic_ai_hybrid_b200.serving import Generator, compute_weights, load_weights  # noqa: E402


def parse(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--preset", default="tiny")
    ap.add_argument("--config", default=None, help="YAML {preset:, overrides:} (atomic_ai_hybrid_b200/configs/)")
    ap.add_argument("--layers", type=int, default=None, help="override the number of layers")
    ap.add_argument("--ckpt-root", default=None)
    ap.add_argument("--ckpt-slot", default="latest")
    ap.add_argument("--ckpt-step", type=int, default=None)
    ap.add_argument("--prompt", action="append", default=[], help="comma-separated token ids (repeatable)")
    ap.add_argument("--prompt-file", default=None)
    ap.add_argument("--prefix", default=None, help="comma-separated token ids before every prompt")
    ap.add_argument("--score", type=int, default=None, metavar="N", help="score the prompts, with N alternatives (0 to 64)")
    ap.add_argument("--kv-budget", type=int, default=0, help="attention rows a head that a conversation is cut back to when its "
                    "--kv-rows run out (0: rows for all its tokens)")
    ap.add_argument("--kv-rows", type=int, default=0, help="attention rows of a conversation (default: prompt and answer)")
    ap.add_argument("--max-new-tokens", type=int, default=32)
    ap.add_argument("--temperature", type=float, default=1.0, help="0: the most likely token")
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--min-p", type=float, default=0.0)
    ap.add_argument("--stop-token", type=int, default=None)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--no-graph", action="store_true", help="launch every token step's kernels one by one")
    return ap.parse_args(argv)


def main(argv=None) -> None:
    a = parse(argv)
    cfg = load_yaml_config(a.config) if a.config else get_preset(a.preset)
    if a.layers is not None:
        cfg = cfg.replace(num_layers=a.layers)
        cfg.validate()
    lines = list(a.prompt)
    if a.prompt_file:
        with open(a.prompt_file) as f:
            lines += [line for line in f.read().splitlines() if line.strip()]
    prompts = [[int(t) for t in line.split(",")] for line in lines]
    prefix = [int(t) for t in a.prefix.split(",")] if a.prefix else None
    bad = [t for p in prompts + [prefix or []] for t in p if not 0 <= t < cfg.vocab_size]
    if not prompts or bad:
        raise SystemExit(f"token ids must lie in [0, {cfg.vocab_size}): {bad[:5]}" if bad else "give --prompt or --prompt-file")
    device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    torch.manual_seed(a.seed)
    with torch.device(device):
        model = HybridMoEModel(cfg, compute_dtype=torch.bfloat16 if device.type == "cuda" else torch.float32)
    if a.ckpt_root:
        absent = load_weights(model, a.ckpt_root, a.ckpt_slot, a.ckpt_step)
        if absent:
            raise SystemExit(f"the checkpoint is of another model, without {', '.join(absent[:8])}")
    most, before = max(map(len, prompts)) + a.max_new_tokens, len(prefix or [])
    gen = Generator(compute_weights(model), len(prompts) + (prefix is not None), max_len=max(a.kv_rows or most, before),
                    cuda_graph=not a.no_graph, max_positions=before + most, kv_budget=a.kv_budget)
    if a.score is not None:
        out = gen.score(prompts, top=a.score, temperature=a.temperature, prefix=prefix)
        for i, p in enumerate(prompts):
            print(json.dumps({"prompt": p, **{name: v[i] for name, v in out.items()}}))
        return
    began = time.perf_counter()
    tokens, logprobs = gen.generate(prompts, a.max_new_tokens, a.temperature, a.top_k, a.top_p, a.min_p, a.stop_token,
                                    torch.Generator(device=device).manual_seed(a.seed), prefix)
    took = time.perf_counter() - began
    for p, t, lp in zip(prompts, tokens, logprobs):
        print(json.dumps({"prompt": p, "tokens": t, "logprobs": [round(x, 5) for x in lp]}))
    n = sum(map(len, tokens))
    print(f"[generate] {n} tokens in {took:.2f} s ({n / took:.1f} tokens/s, prompts and graph capture included)", file=sys.stderr)


if __name__ == "__main__":
    main()
