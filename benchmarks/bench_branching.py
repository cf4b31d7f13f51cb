"""Steps of the Llama-3-8B shape that carry several continuations: beams, and trees of drafts, beside plain decode steps and chains of drafts.

    python benchmarks/bench_branching.py [--context 1500] [--beams 4 16] [--trees 1x13 1x33 16x13]

Random weights, random prompts. Prints the milliseconds of a step through the engine, host included (median of 5 rounds of 10 steps): a decode step, a beam step (forward of all beams, choice of the
continuations, reordering), the verification of a chain of drafts, and that of a tree of as many (forward, picks, acceptance)."""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from benchmarks.bench_page_budget import LLAMA3_8B  # noqa: E402


def median_ms(step, rounds=5, steps=10) -> float:
    for _ in range(3):
        step()
    times = []
    for _ in range(rounds):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(steps):
            step()
        torch.cuda.synchronize()
        times.append((time.perf_counter() - t) / steps * 1e3)
    return sorted(times)[rounds // 2]


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--context", type=int, default=1500)
    ap.add_argument("--beams", type=int, nargs="+", default=[4, 16])
    ap.add_argument("--trees", nargs="+", default=["1x13", "1x33", "16x13"], help="sequences x tokens of a tree")
    args = ap.parse_args()
    from inference_b200 import ops
    from inference_b200.engine.backend import GpuBackend
    from inference_b200.engine.branching import best_continuations
    from inference_b200.engine.llm_engine import EngineConfig, LlmEngine
    from inference_b200.models import ModelConfig
    from inference_b200.models.llama import LlamaGpu

    room = -(-(args.context + 1024) // 1024) * 1024
    cfg = ModelConfig.from_json(dict(LLAMA3_8B, max_position_embeddings=room))
    eng = LlmEngine(LlamaGpu(cfg, device=torch.device("cuda")).init_random(seed=0), EngineConfig(max_batch=32, max_seq_len=room))
    be = GpuBackend(eng.runner)
    draw = lambda n: torch.randint(0, cfg.vocab_size, (n,)).tolist()

    def prompts(n):
        seqs = [be.new_sequence() for _ in range(n)]
        for s in seqs:
            be.forward([s], [draw(args.context)])
        return seqs

    def decode_ms(n):
        seqs = prompts(n)
        ms = median_ms(lambda: be.forward_greedy(seqs, [[1]] * n))
        for s in seqs:
            be.release(s)
        return ms

    for beams in args.beams:
        state = {"seqs": be.reorder(prompts(1), [0] * beams), "tokens": [1] * beams, "scores": [-float(i) for i in range(beams)]}

        def step():
            rows = be.forward(state["seqs"], [[t] for t in state["tokens"]])
            best = best_continuations(torch.stack(list(rows)), torch.tensor(state["scores"]).cuda(), 2 * beams)[:beams]
            state["scores"], state["tokens"] = [s for s, _, _ in best], [t for _, _, t in best]
            state["seqs"] = be.reorder(state["seqs"], [b for _, b, _ in best])

        ms = median_ms(step)
        for s in state["seqs"]:
            be.release(s)
        print(f"{beams} beams: {ms:.2f} ms a step; {beams} sequences decoded greedily: {decode_ms(beams):.2f}", flush=True)
    for shape in args.trees:
        n, size = map(int, shape.split("x"))
        parents = [[-1] + [(i - 1) // 2 for i in range(1, size)]] * n
        drafts = [draw(size) for _ in range(n)]
        seqs = prompts(n)

        def tree():
            be.step_trees(seqs, drafts, parents, ops.argmax)
            for s in seqs:
                be.truncate(s, args.context)

        def chain():
            rows = be.forward(seqs, drafts, all_positions=True)
            ops.argmax(torch.cat(rows)).tolist()
            for s in seqs:
                be.truncate(s, args.context)

        print(f"{n} x {size} drafts behind {args.context} tokens: {median_ms(tree):.2f} ms as trees, {median_ms(chain):.2f} as chains, {decode_ms(n):.2f} a decode step", flush=True)
        for s in seqs:
            be.release(s)


if __name__ == "__main__":
    main()
