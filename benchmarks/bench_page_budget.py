"""Decode steps of the Llama-3-8B shape over long contexts, all of them against a page budget.

    python benchmarks/bench_page_budget.py [--pages 128] [--shape 8x30000 1x30000 32x8000]

Random weights and random cached keys and values, contexts in a paged cache of 16-token pages; a budget of N pages reads the first one, the last four and the best N - 5 of
the others. Prints the milliseconds of a step from its captured graph, host included (median of 5 rounds of 20 steps behind 5 of warm-up)."""
import argparse
import gc
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

LLAMA3_8B = {"architectures": ["LlamaForCausalLM"], "hidden_size": 4096, "intermediate_size": 14336, "num_hidden_layers": 32, "num_attention_heads": 32,
             "num_key_value_heads": 8, "vocab_size": 128256, "rms_norm_eps": 1e-5, "rope_theta": 500000.0, "tie_word_embeddings": False}


def step_ms(batch: int, context: int, budget) -> float:
    from inference_b200 import ops
    from inference_b200.engine.llm_engine import EngineConfig, LlmEngine
    from inference_b200.models import ModelConfig
    from inference_b200.models.llama import LlamaGpu

    room = -(-(context + 256) // 1024) * 1024
    cfg = ModelConfig.from_json(dict(LLAMA3_8B, max_position_embeddings=room))
    eng = LlmEngine(LlamaGpu(cfg, device=torch.device("cuda")).init_random(seed=0), EngineConfig(max_batch=batch, max_seq_len=room, page_budget=budget))
    g = torch.Generator(device="cuda").manual_seed(1)
    for layer in eng.pool.data:
        layer.copy_(torch.randn(layer.shape, device="cuda", dtype=layer.dtype, generator=g))
    seqs = [eng.new_sequence() for _ in range(batch)]
    for s in seqs:
        s.reserve(context)
    if budget is not None:
        table, lens = torch.tensor([s.blocks for s in seqs], dtype=torch.int32, device="cuda"), torch.full((batch,), context, dtype=torch.int32, device="cuda")
        for layer, sums in zip(eng.pool.data, eng.pool.summaries):
            ops.summarize_pages(layer[0], table, lens, sums, cu_q=None, max_q_len=context)
    for _ in range(5):
        eng.runner.decode(seqs, [1] * batch)
    rounds = []
    for _ in range(5):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(20):
            eng.runner.decode(seqs, [1] * batch)
        torch.cuda.synchronize()
        rounds.append((time.perf_counter() - t) / 20 * 1e3)
    return sorted(rounds)[2]


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--pages", type=int, default=128, help="pages that a token reads")
    ap.add_argument("--shape", nargs="+", default=["8x30000", "1x30000", "32x8000"], help="sequences x tokens in each")
    args = ap.parse_args()
    from inference_b200 import ops

    for shape in args.shape:
        batch, context = map(int, shape.split("x"))
        times = []
        for budget in (None, ops.PageBudget(top=args.pages - 5)):
            times.append(step_ms(batch, context, budget))
            gc.collect()
            torch.cuda.empty_cache()
        print(f"{batch} x {context} tokens: {times[0]:.2f} ms a step over all of them, {times[1]:.2f} ms over {args.pages} pages each", flush=True)


if __name__ == "__main__":
    main()
