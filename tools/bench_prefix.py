"""Several questions about one clip, and bounded caches, at Vicuna-7B shape (random weights): prefill and decode step of a batch whose prompts
begin alike, with the shared rows in every sequence's prompt and once (make_prefix / prefill(prefix=) / generate(prefix=)); decode step with
the whole cache and with one cut to a budget (generate(cache_budget=)).  python tools/bench_prefix.py"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from hawkeye_amd.config import VICUNA_7B  # noqa: E402
from hawkeye_amd.decode import LlamaGenerator  # noqa: E402
from hawkeye_amd.llm import LlamaPrefill  # noqa: E402


def ms(f, n):
    f()
    f()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(n):
        f()
    torch.cuda.synchronize()
    return (time.perf_counter() - t0) * 1e3 / n


def main():
    dev = "cuda"
    pre = LlamaPrefill(VICUNA_7B, dev).init_random(0)
    gen = LlamaGenerator(pre)
    V = VICUNA_7B.vocab_size
    for B, P, S in ((4, 352, 37), (8, 352, 37), (8, 1500, 37), (16, 1500, 37)):
        shared, own = torch.randint(0, V, (1, P), device=dev), torch.randint(0, V, (B, S), device=dev)
        full = torch.cat([shared.expand(B, P), own], 1)
        pf = pre.make_prefix(src=shared)
        m = ms(lambda: pre.make_prefix(src=shared), 5)
        a, b = ms(lambda: pre.prefill(src=full), 5), ms(lambda: pre.prefill(src=own, prefix=pf), 5)
        ga, gb = ms(lambda: gen.generate(src=full, max_new_tokens=21), 2), ms(lambda: gen.generate(src=own, prefix=pf, max_new_tokens=21), 2)
        print(f"{B} prompts of {P} shared + {S} own tokens: prefill {a:.2f} ms -> {m:.2f} (shared, once) + {b:.2f}; "
              f"step {(ga - a) / 20:.3f} ms -> {(gb - b) / 20:.3f}", flush=True)
    for B, S, budget in ((1, 1500, 256), (8, 1500, 256), (16, 1500, 256)):
        src = torch.randint(0, V, (B, S), device=dev)
        whole = [ms(lambda: gen.generate(src=src, max_new_tokens=n), 2) for n in (11, 51)]
        cut = [ms(lambda: gen.generate(src=src, max_new_tokens=n, cache_budget=budget), 2) for n in (11, 51)]
        print(f"{B} prompts of {S} tokens, budget {budget}: prompt and 11 tokens {whole[0]:.2f} ms -> {cut[0]:.2f}; "
              f"step {(whole[1] - whole[0]) / 40:.3f} ms -> {(cut[1] - cut[0]) / 40:.3f}", flush=True)


if __name__ == "__main__":
    main()
