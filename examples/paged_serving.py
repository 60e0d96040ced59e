"""A serving loop over the paged 4-bit cache (mlops_b200.attention.paged): requests of different lengths arrive, their prompts are processed together, then
every request gets one token per step, the step captured into a CUDA graph.

    python examples/paged_serving.py [--requests 8] [--steps 64] [--prompt 1500]

The model is left out: queries, keys and values are random numbers where an engine has its projections. What an engine keeps between the steps is here: a pool of
pages per layer, one block table, the requests' lengths, the ring of free pages and its two ends, all on the GPU.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from mlops_b200.attention import paged  # noqa: E402

Q_HEADS, KV_HEADS, PAGE = 32, 8, 64


def rows(tokens, generator):
    """queries, keys and values of `tokens` tokens as slices of a fused projection's rows"""
    x = torch.randn((tokens, Q_HEADS + 2 * KV_HEADS, 128), generator=generator, device="cuda").to(torch.bfloat16)
    return x.split([Q_HEADS, KV_HEADS, KV_HEADS], 1)


def serve(requests=8, steps=64, prompt=1500, seed=0):
    """Returns the lengths at the end, the last step's outputs and the seconds that the decode steps took."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    prompts = [1 + (prompt * (i + 1)) // requests for i in range(requests)]
    width = -(-(max(prompts) + steps) // PAGE)
    pages = sum(-(-(n + steps) // PAGE) for n in prompts)
    cache = paged.empty(pages, KV_HEADS, PAGE, v_scale=torch.full((KV_HEADS,), 0.5))
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")
    free = torch.arange(pages, dtype=torch.int32, device="cuda")
    cursor = torch.tensor([0, pages, 0], dtype=torch.int64, device="cuda")

    # the prompts, all in one step
    added = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    q, k, v = rows(sum(prompts), generator)
    step = paged.assign(table, lengths, added, free, cursor, PAGE, sum(prompts))
    paged.append(cache, k, v, step.slots)
    paged.attend(q, cache, table, step.lengths, step.starts)
    lengths.copy_(step.lengths)
    cursor.copy_(step.cursor)

    # one token per request and step: pages, append, attention as one graph, which finds the lengths that the last replay left
    one = torch.ones_like(lengths)
    q, k, v = (x.contiguous() for x in rows(requests, generator))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = paged.assign(table, lengths, one, free, cursor, PAGE, requests)
        paged.append(cache, k, v, step.slots)
        out = paged.attend(q, cache, table, step.lengths)
        lengths.copy_(step.lengths)
        cursor.copy_(step.cursor)
    torch.cuda.synchronize()
    begin = time.perf_counter()
    for _ in range(steps):
        for x, new in zip((q, k, v), rows(requests, generator)):
            x.copy_(new)
        graph.replay()
    torch.cuda.synchronize()
    seconds = time.perf_counter() - begin
    if int(cursor[2]):
        raise RuntimeError(f"{int(cursor[2])} pages were missing")
    return lengths.tolist(), out, seconds


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--requests", type=int, default=8)
    parser.add_argument("--steps", type=int, default=64)
    parser.add_argument("--prompt", type=int, default=1500)
    args = parser.parse_args()
    lengths, out, seconds = serve(args.requests, args.steps, args.prompt)
    print(f"{args.requests} requests of {min(lengths)} to {max(lengths)} tokens, {args.steps} steps: {seconds / args.steps * 1e6:.1f} us per step, "
          f"{args.requests * args.steps / seconds:.0f} tokens/s, largest output {out.abs().max().item():.3f}")


if __name__ == "__main__":
    main()
