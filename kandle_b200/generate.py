"""Generation from a checkpoint folder:

    python -m kandle_b200.generate --model DIR --prompt "5 17 3" [--steps 32] [--dtype bfloat16|float32]
                                   [--temperature T --top-k K --top-p P --seed S] [--beams N [--eos ID] [--length-penalty P]]

The model class follows from config.json (kandle_b200.registry).  Prompts are token ids (this package has no
tokenizer); several --prompt of one length run as a batch.  Prints the generated ids, one line a prompt
(with --beams the best hypothesis of a beam search).
"""
from __future__ import annotations

import argparse

import numpy as np


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="python -m kandle_b200.generate", description="Generates tokens from a checkpoint folder.")
    ap.add_argument("--model", required=True, help="folder with config.json and model.safetensors")
    ap.add_argument("--prompt", required=True, action="append", help="token ids; repeat for a batch of equal lengths")
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float32"])
    ap.add_argument("--temperature", type=float, default=None, help="sample instead of the greedy choice")
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--beams", type=int, default=0, help="beam search with this many beams (Qwen3)")
    ap.add_argument("--eos", type=int, default=-1, help="token that ends a hypothesis of the beam search")
    ap.add_argument("--length-penalty", type=float, default=1.0)
    a = ap.parse_args(argv)
    if a.beams < 0 or (a.beams and a.temperature is not None):
        ap.error("--beams takes a positive number and no --temperature")
    rows = [[int(x) for x in p.split()] for p in a.prompt]
    if len({len(r) for r in rows}) != 1 or not rows[0]:
        ap.error("prompts must have one length, at least one token")
    import kandle_b200
    from . import registry
    kandle_b200.init(0)
    if a.beams:
        if registry.lookup(registry.load_config(a.model)) is not registry.lookup({"architectures": ["Qwen3ForCausalLM"]}):
            ap.error("--beams: this architecture's engine has no beam search")
        n = len(rows) * a.beams
        engine = registry.load_engine(a.model, n, len(rows[0]) + a.steps, a.dtype, paged=True, spare_pages=2 * n)
        for hypotheses in engine.generate_beams(np.asarray(rows, np.int32), a.beams, a.steps, a.eos, a.length_penalty):
            print(" ".join(str(t) for t in hypotheses[0][0]))
        engine.dispose()
        return 0
    engine = registry.load_engine(a.model, len(rows), len(rows[0]) + a.steps, a.dtype)
    if a.temperature is not None:
        engine.set_sampler(a.temperature, a.top_k, a.top_p, a.seed)
    for row in engine.generate(np.asarray(rows, np.int32), a.steps):
        print(" ".join(str(t) for t in row))
    engine.dispose()
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
