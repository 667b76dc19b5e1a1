"""Command line of the serving path.

    python -m krasis_b200 generate --model DIR --prompt-ids 5,17,3 [--prompt-ids ...] [--max-new-tokens 32] [--dtype bfloat16]
                                   [--temperature 0 --top-k 0 --top-p 1 --seed 0] [--max-tokens 8192] [--step-tokens 512]
                                   [--logprobs N] [--expert-format e4m3]
    python -m krasis_b200 score    --model DIR --prompt-ids 5,17,3 [--prompt-ids ...] [--dtype bfloat16] [--max-tokens 8192] [--step-tokens 512]
                                   [--expert-format e4m3]
    python -m krasis_b200 trace    --model DIR --dtype bfloat16|float32 --out DIR --max-tokens N        (same as bin/trace_run)

`generate` loads the checkpoint through the model registry (config.json decides the class), runs continuous batching over the
given prompts and prints one JSON line per prompt with the generated token ids (and, with --logprobs, the log probability and entropy of each
and the N most likely tokens).  `score` prints the log probabilities of the given tokens, each after those before it, and the perplexity;
numbers that JSON does not have (the log probability of a token that cannot be, a perplexity beyond a double, NaN) are null.  Token ids in, token ids out: tokenisers are not
part of this package."""
import argparse
import json
import math
import sys


def perplexity(logprobs):
    """exp of minus the mean; None of nothing, inf of what passes a double."""
    if not logprobs:
        return None
    mean = -sum(logprobs) / len(logprobs)
    return math.inf if mean > 709 else math.exp(mean)


def json_line(record) -> str:
    """One line of JSON; numbers that it cannot hold (infinities, NaN) are null."""
    def held(x):
        if isinstance(x, dict):
            return {k: held(v) for k, v in x.items()}
        if isinstance(x, (list, tuple)):
            return [held(v) for v in x]
        return None if isinstance(x, float) and not math.isfinite(x) else x
    return json.dumps(held(record), allow_nan=False)


def main(argv=None) -> int:
    argv = sys.argv[1:] if argv is None else argv
    if argv and argv[0] == "trace":
        from .trace_runner import main as trace_main
        return trace_main(argv[1:])
    ap = argparse.ArgumentParser(prog="python -m krasis_b200", description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("command", choices=["generate", "score"])
    ap.add_argument("--model", required=True)
    ap.add_argument("--prompt-ids", action="append", required=True, help="comma-separated token ids; repeat for several prompts")
    ap.add_argument("--max-new-tokens", type=int, default=32)
    ap.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float32"])
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--seed", type=int, default=None)
    ap.add_argument("--eos", type=int, default=None)
    ap.add_argument("--max-tokens", type=int, default=8192, help="tokens the cache pool holds")
    ap.add_argument("--max-requests", type=int, default=4)
    ap.add_argument("--step-tokens", type=int, default=512, help="token budget of one step (prompt portions + decoded tokens)")
    ap.add_argument("--expert-format", default=None, choices=["e4m3"], help="routed experts held in 8-bit floating point (Megolorn, without identity experts)")
    ap.add_argument("--logprobs", type=int, default=None, help="log probabilities of the generated tokens, with this many alternatives (0 to 64)")
    a = ap.parse_args(argv)

    import torch
    from .registry import check_expert_format, load_model
    from .sampling import SamplingParams
    from .scheduler import Scheduler
    from .seqops import MAX_TOP_LOGPROBS
    if a.logprobs is not None and not 0 <= a.logprobs <= MAX_TOP_LOGPROBS:
        ap.error(f"--logprobs {a.logprobs}: 0 to {MAX_TOP_LOGPROBS} alternatives")
    if a.command == "score" and a.step_tokens < 1:
        ap.error(f"--step-tokens {a.step_tokens}: portions of at least one token")
    if a.expert_format:
        try:
            check_expert_format(a.model, a.expert_format)
        except ValueError as e:
            print(e, file=sys.stderr)
            return 3
    model = load_model(a.model, dtype=torch.bfloat16 if a.dtype == "bfloat16" else torch.float32, **({"expert_format": a.expert_format} if a.expert_format else {}))
    if not hasattr(model, "forward_step"):
        print(f"{type(model).__name__} has no step interface for generation", file=sys.stderr)
        return 3
    prompts = [[int(t) for t in p.split(",") if t.strip()] for p in a.prompt_ids]
    sched = Scheduler(model, max_tokens=a.max_tokens, max_requests=a.max_requests, cuda_graphs=True)
    if a.command == "score":
        for p, s in zip(prompts, sched.score(prompts, step_tokens=a.step_tokens)):
            print(json_line({"prompt_tokens": len(p), "logprobs": s, "perplexity": perplexity(s)}))
        return 0
    outs = sched.generate(prompts, a.max_new_tokens, SamplingParams(a.temperature, a.top_k, a.top_p, a.seed), step_tokens=a.step_tokens,
                          eos=a.eos, logprobs=a.logprobs)
    told = [{}] * len(prompts)
    if a.logprobs is not None:
        outs, details = outs
        told = [{"logprobs": d} for d in details]
    for p, o, d in zip(prompts, outs, told):
        print(json_line({"prompt_tokens": len(p), "generated": o, **d}))
    return 0


if __name__ == "__main__":
    sys.exit(main())
