"""Command line: greedy generation from token ids with any model the registry knows, log probabilities of given
continuations with the factorized decoder.

    python -m quantibbler_b200 generate --model DIR --prompt 5,17,3 --max-tokens 32
    python -m quantibbler_b200 score --model DIR --prompt 5,17,3 --continuation 9,2 --continuation 4 --top 5
    python -m quantibbler_b200 trace --model DIR --out OUT < steps.jsonl

Prints one JSON object (token ids in and out: text needs the model's tokenizer, which is not part
of this package)."""

from __future__ import annotations

import argparse
import json
import sys


def main(argv=None) -> int:
    argv = sys.argv[1:] if argv is None else argv
    if argv[:1] == ["trace"]:
        from .trace import main as trace_main
        return trace_main(argv[1:])
    ap = argparse.ArgumentParser(prog="quantibbler_b200")
    sub = ap.add_subparsers(dest="command", required=True)
    g = sub.add_parser("generate", help="greedy continuation of a prompt")
    g.add_argument("--model", required=True, help="a folder with config.json, a model directory or a blob")
    g.add_argument("--prompt", required=True, help="token ids, with commas between them")
    g.add_argument("--max-tokens", type=int, default=32)
    g.add_argument("--eos", type=int, default=None, help="token id that ends the generation")
    g.add_argument("--dtype", choices=("bfloat16", "float32"), default=None, help="default: the model's own")
    g.add_argument("--kv-dtype", choices=("bfloat16", "float32", "int8"), default=None,
                   help="storage of the key/value cache (factorized decoder; default: the model's own)")
    sc = sub.add_parser("score", help="log probabilities of continuations of a prompt")
    sc.add_argument("--model", required=True, help="a model directory or a blob")
    sc.add_argument("--prompt", required=True, help="token ids, with commas between them")
    sc.add_argument("--continuation", required=True, action="append", help="token ids; may be given several times")
    sc.add_argument("--top", type=int, default=0, help="most probable alternatives to print at each place")
    sc.add_argument("--dtype", choices=("bfloat16", "float32"), default=None, help="default: the model's own")
    sc.add_argument("--kv-dtype", choices=("bfloat16", "float32", "int8"), default=None,
                    help="storage of the key/value cache (default: float32, the slowest by far)")
    sub.add_parser("trace", help="replay a trace of token ids (see bin/trace_run)")
    a = ap.parse_args(argv)
    from .gpu import GpuContext
    from .registry import UnknownSetting, load_decoder
    prompt = [int(t) for t in a.prompt.split(",")]
    settings = {} if a.dtype is None else {"serving": a.dtype}
    if a.kv_dtype is not None:
        settings["kv_dtype"] = a.kv_dtype
    if a.command == "score":
        conts = [[int(t) for t in c.split(",")] for c in a.continuation]
        settings.update(max_batch=len(conts), max_prefix=len(prompt), max_seq=max(len(c) for c in conts))
    else:
        settings["max_seq"] = len(prompt) + max(a.max_tokens, 1)
    try:
        decoder = load_decoder(GpuContext.init(), a.model, **settings)
    except UnknownSetting as e:   # (--kv-dtype or score with a model of another kind)
        ap.error(str(e))
    print(json.dumps(decoder.score(prompt, conts, a.top) if a.command == "score" else
                     decoder.generate(prompt, a.max_tokens, a.eos)))
    return 0


if __name__ == "__main__":
    sys.exit(main())
