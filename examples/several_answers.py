"""Several answers to one prompt, with weights, keys and values in 4 bits.

    python examples/several_answers.py -m MODEL_DIR -p 2,651,1234 --answers 4 -n 32 --temp 0.8
    python examples/several_answers.py --random config.json -p 2,651,1234          # random weights

The prompt is run once; the conversations forked from it share its pages and copy one only when they write into it.  Then the
cache is made as small as what is left needs.
"""
from __future__ import annotations

import argparse
import json
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("-m", "--model")
    ap.add_argument("--random", help="a config.json: random weights instead of a model folder")
    ap.add_argument("-p", "--prompt", required=True, help="token ids separated by commas")
    ap.add_argument("-n", type=int, default=32)
    ap.add_argument("--answers", type=int, default=4)
    ap.add_argument("--temp", type=float, default=0.8)
    ap.add_argument("--seed", type=int, default=42)
    ap.add_argument("--max-seq-len", type=int, default=4096)
    a = ap.parse_args(argv)
    from hos_b200 import Engine
    from hos_b200.registry import config_from_dict
    prompt = [int(t) for t in a.prompt.split(",")]
    how = dict(max_batch=a.answers + 1, max_seq_len=a.max_seq_len, weight_bits=4, cache_bits=4)
    if a.random:
        with open(a.random) as f:
            eng = Engine.from_config(config_from_dict(json.load(f)), seed=a.seed, **how)
    else:
        eng = Engine(a.model, **how)
    first, = eng.open(1)
    if len(prompt) > 1:
        eng.step([first.slot], [prompt[:-1]])           # all of the prompt but its last token, which every answer runs for itself
        first.position = len(prompt) - 1
    first.pending = prompt[-1]
    chats = [first] + first.fork(a.answers - 1)
    for answer in eng.generate_from_ids(chats, [[] for _ in chats], max_tokens=a.n, temp=a.temp, seed=a.seed):
        print(",".join(map(str, answer)))
    for c in chats[1:]:
        c.close()
    cache = eng.runner.cache
    eng.runner.resize_cache(max(64, first.position + a.n))
    print(f"[hos] {cache.bytes_per_token()} bytes of keys and values a token, {cache.tokens_capacity()} tokens of cache left", file=sys.stderr)
    first.close()
    return 0


if __name__ == "__main__":
    sys.exit(main())
