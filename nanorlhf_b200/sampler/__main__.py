"""Generate from a checkpoint folder with the in-process rollout engine of its model family.

    python -m nanorlhf_b200.sampler --model DIR --prompt-ids 5,17,3 [--prompt-ids ...] [--n 1] [--max-tokens 32]
                                    [--temperature 0] [--top-p 1.0] [--top-k 0] [--min-p 0] [--seed 0] [--dtype bfloat16|float32] [--eos -1]
                                    [--shared-decode | --kv-budget 0 [--kv-sinks 4] [--kv-recent N]]

The model class and its engine (whole-prompt paged-KV engine or the step engine of hybrid decoders) are chosen by
``config.json``.  Prints one JSON line per sample: {"prompt": i, "sample": j, "tokens": [...]}.
"""
import argparse
import json
import sys


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--model", required=True)
    ap.add_argument("--prompt-ids", action="append", required=True, help="comma-separated token ids; repeat for more prompts")
    ap.add_argument("--n", type=int, default=1)
    ap.add_argument("--max-tokens", type=int, default=32)
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--top-k", type=int, default=0, help="0: off")
    ap.add_argument("--min-p", type=float, default=0.0, help="0: off")
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float32"])
    ap.add_argument("--eos", type=int, default=-1, help="stop token id (-1: none)")
    ap.add_argument("--pad", type=int, default=0)
    ap.add_argument("--shared-decode", action="store_true", help="read the prompt pages that samples share once for all of them")
    ap.add_argument("--kv-budget", type=int, default=0, help="cached tokens that a sample goes back to every 64 steps (0: all stay)")
    ap.add_argument("--kv-sinks", type=int, default=4, help="first tokens that an eviction keeps")
    ap.add_argument("--kv-recent", type=int, default=None, help="newest tokens that it keeps (a quarter of the budget)")
    a = ap.parse_args()
    import torch
    from ..csrc.build import build
    build(verbose=False)
    from ..models.registry import load_model, sampler_kind
    from .engine import generate

    class _Tok:                                   # the engine only needs the two special ids
        pad_token_id, eos_token_id = a.pad, (a.eos if a.eos >= 0 else None)

    dev = torch.device("cuda:0")
    model = load_model(a.model, torch.float32 if a.dtype == "float32" else torch.bfloat16, dev)
    prompts = [[int(t) for t in p.split(",")] for p in a.prompt_ids]
    kw = {"rollout_dtype": a.dtype} if sampler_kind(model) == "hybrid" else {}
    out = generate(a.n, model, _Tok, prompts, a.temperature, a.max_tokens, top_p=a.top_p, seed=a.seed, backend="native",
                   eos_token_id=a.eos, top_k=a.top_k, min_p=a.min_p,
                   shared_decode=a.shared_decode, kv_budget=a.kv_budget, kv_sinks=a.kv_sinks, kv_recent=a.kv_recent, **kw).tolist()
    for i in range(len(prompts)):
        for j in range(a.n):
            print(json.dumps({"prompt": i, "sample": j, "tokens": out[i * a.n + j]}))
    return 0


if __name__ == "__main__":
    sys.exit(main())
