"""A request's life with the paged cache: audit in 16 bits, decode from 4-bit pages, audit again.

    python -m code_for_iclr27_b200.paged_example [--layers L] [--rows N] [--steps S] [--bits 4|16] [--group G]

A synthetic request's packed cache is audited and evicted (audit.audit_pass), its surviving rows go into pages
(PagedCache.load), decode steps append the new token's rotated, quantised rows and attend over the pages, and the rows
come back into the packed layout (to_packed) for the next audit.  The same steps on 16-bit pages, on the same inputs,
show what 4 bits cost.  Returns (and prints) the bytes a row takes, the device's time of a step's appends and attentions
(the host's page allocation, PagedCache.advance, comes before it) and how far the outputs are off.
"""
from __future__ import annotations

import argparse
import sys


def run(layers: int = 4, heads: int = 8, groups: int = 4, dim: int = 128, rows: int = 4096, steps: int = 16, bits: int = 4,
        group: int = 64, page_size: int = 64, seed: int = 0) -> dict:
    import torch

    from .audit import audit_pass
    from .kvcache import PackedCache
    from .paged import PagedCache, rotary_table

    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, scale=1.0):
        return (scale * torch.randn(shape, generator=g, device=device)).to(dtype)

    # The request after its prefill: every head holds the prompt and some generated rows.
    packed, prompt = PackedCache(), rows * 3 // 4
    for _ in range(layers):
        positions = torch.arange(rows, dtype=torch.float32, device=device).repeat(heads)
        packed.add_layer(normal(heads * rows, dim), normal(heads * rows, dim), positions, [rows] * heads, [prompt] * heads)
    packed.seen_tokens = rows

    # Audit: score the generated rows by the last queries, evict the least needed.
    window = 32
    queries = [normal(window, heads * groups, dim) for _ in range(layers)]
    gradients = [normal(heads * groups, dim, dtype=torch.float32, scale=dim ** -0.5) for _ in range(layers)]
    at = torch.arange(rows - window, rows, device=device)
    margin = torch.tensor([0.7], device=device)
    evicted = layers * heads * rows // 16
    audit_pass(packed, queries, at, gradients, margin, immediate=evicted, queued=0)

    # Decode from pages: 16 bits beside the asked-for form, on the same inputs.
    need = sum(-(-(n + steps) // page_size) for layer in packed.layers for n in layer.head_lens)
    caches = [PagedCache(layers, 1, heads, dim, need, device, torch.bfloat16, b, group, page_size, rows + steps + page_size)
              for b in (16, bits)]
    for cache in caches:
        cache.load(0, packed)
    rotary = rotary_table(rows + steps, dim, 500000.0, device)
    worst, times = 0.0, [[], []]
    for step in range(steps):
        joint = [normal(1, (groups + 2) * heads, dim) for _ in range(layers)]  # each layer's projection of the token
        position = torch.full((1,), packed.seen_tokens + step, device=device)
        outs = []
        for index, cache in enumerate(caches):
            cache.advance([1])
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for layer in range(layers):
                q, k, v = joint[layer].split([groups * heads, heads, heads], 1)
                turned = cache.append(layer, k, v, position, rotary, queries=q)
                out, _ = cache.attend(layer, turned)
            end.record()
            outs.append(out.float())
            times[index].append((begin, end))
        worst = max(worst, float((outs[1] - outs[0]).norm() / outs[0].norm()))
    torch.cuda.synchronize()
    for cache in caches:
        cache.check_flags()

    # The next audit works on the packed layout again.
    back = caches[1].to_packed(0)
    audit_pass(back, queries, at, gradients, margin, immediate=layers * heads, queued=0)
    caches[1].load(0, back)
    middle = [sorted(b.elapsed_time(e) * 1e3 for b, e in t)[len(t) // 2] for t in times]
    row_bytes = [2 * 2 * dim, 2 * (dim // 2 + 4 * dim // group) if bits == 4 else 2 * 2 * dim]
    return {"rows": int(caches[0].rows.sum()), "evicted": evicted, "row_bytes_16": row_bytes[0], "row_bytes": row_bytes[1],
            "step_us_16": middle[0], "step_us": middle[1], "relative_error": worst,
            "rows_after_audit": int(caches[1].rows.sum())}


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--layers", type=int, default=4)
    parser.add_argument("--rows", type=int, default=4096)
    parser.add_argument("--steps", type=int, default=16)
    parser.add_argument("--bits", type=int, default=4, choices=(4, 16))
    parser.add_argument("--group", type=int, default=64, choices=(32, 64, 128))
    args = parser.parse_args(argv)
    result = run(args.layers, rows=args.rows, steps=args.steps, bits=args.bits, group=args.group)
    print(f"{result['rows']} rows in pages after the audit evicted {result['evicted']}; a row takes {result['row_bytes']} "
          f"bytes ({result['row_bytes_16']} in 16 bits)")
    print(f"step over {args.layers} layers: {result['step_us']:.1f} us ({result['step_us_16']:.1f} us from 16-bit pages); "
          f"outputs differ by {result['relative_error']:.4f} of their norm")
    print(f"{result['rows_after_audit']} rows after the next audit")


if __name__ == "__main__":
    sys.exit(main())
