"""Serving long requests from the 4-bit latent cache: prefill, then decode over all pages or over chosen ones.

Synthetic latents (512 wide, rotary part 64, 16 heads) are stored for a
few ragged requests; then tokens are decoded step by step, the same ones in two ways: attention over every page, and
over the ``budget`` pages a request whose boxes score highest.  A step stores its tokens' rows, refreshes the boxes of the
pages they fell into and attends, layer by layer; both ways are captured in a CUDA graph each and replayed.

    python examples/int4_long_context.py [--requests 32] [--context 32768] [--budget 32] [--layers 2] [--steps 16]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from mla_kv_quant_b200 import int4  # noqa: E402


def run(requests: int = 32, context: int = 32768, budget: int = 32, layers: int = 2, steps: int = 16, heads: int = 16,
        d: int = 512, dr: int = 64, seed: int = 0) -> dict:
    """The steps' milliseconds, the last step's outputs, and how far the chosen pages' attention is from the whole one."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    lens = torch.randint(context // 2, context + 1, (requests,), generator=g, device=dev, dtype=torch.int32)
    need = -(-(context + steps) // int4.PAGE)
    pool = int4.Int4LatentPool(size=int4.PAGE * (requests * need + 1), layer_num=layers, kv_lora_rank=d, qk_rope_head_dim=dr,
                               device=dev, boxes=True)
    # pages are dealt in an arbitrary order; page 0 is left to padding
    table = (torch.randperm(requests * need, generator=g, device=dev).to(torch.int32) + 1).view(requests, need)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    sm_scale = (128 + dr) ** -0.5

    def slots_of(request, positions):
        return table[request, positions // int4.PAGE].long() * int4.PAGE + positions % int4.PAGE

    # ---- prefill: a request's rows, then the boxes of its pages ----
    # Each request's tokens drift, so that neighbours are alike and pages differ, as a context's do.
    for b in range(requests):
        n = int(lens[b])
        pos = torch.arange(n, device=dev)
        pages = table[b, : -(-n // int4.PAGE)].contiguous()
        counts = torch.full_like(pages, int4.PAGE)
        counts[-1] = n - (len(pages) - 1) * int4.PAGE
        for layer in range(layers):
            topic = rand(len(pages), d + dr).repeat_interleave(int4.PAGE, 0)[:n]
            rows = topic + 0.5 * rand(n, d + dr)
            pool.write(layer, rows[:, :d].bfloat16(), rows[:, d:].bfloat16(), slots_of(b, pos), err)
            pool.update_boxes(layer, pages, counts, err)

    # ---- decode: buffers that a graph's replays read and write ----
    ws = pool.workspace(requests, heads, need, budget=budget)
    seq_lens, slots = lens.clone(), torch.zeros(requests, dtype=torch.int64, device=dev)
    new_rows = torch.zeros(layers, requests, d + dr, dtype=torch.bfloat16, device=dev)
    q = torch.zeros(layers, requests, heads, d + dr, dtype=torch.bfloat16, device=dev)
    last_pages, last_counts = (torch.zeros(requests, dtype=torch.int32, device=dev) for _ in range(2))
    out = {name: torch.zeros(layers, requests, heads, d, dtype=torch.bfloat16, device=dev) for name in ("all", "chosen")}
    lse = {name: torch.zeros(layers, requests, heads, device=dev) for name in out}

    def step(name):
        for layer in range(layers):
            pool.write(layer, new_rows[layer, :, :d], new_rows[layer, :, d:], slots, err)
            pool.update_boxes(layer, last_pages, last_counts, err)
            if name == "all":
                pool.decode(layer, q[layer], table, seq_lens, sm_scale, out[name][layer], lse[name][layer], ws, err)
            else:
                pool.sparse_decode(layer, q[layer], table, seq_lens, sm_scale, budget, out[name][layer], lse[name][layer], ws,
                                   err=err)

    each = torch.arange(requests, device=dev)

    def next_token():
        pos = seq_lens.long()
        slots.copy_(slots_of(each, pos))
        last_pages.copy_(table[each, pos // int4.PAGE])
        last_counts.copy_(pos % int4.PAGE + 1)
        seq_lens.add_(1)
        new_rows.copy_(rand(layers, requests, d + dr))
        # a query asks for what a place of its request holds
        for layer in range(layers):
            kv, pe = (torch.empty(requests, w, dtype=torch.bfloat16, device=dev) for w in (d, dr))
            at = (torch.rand(requests, generator=g, device=dev) * pos).long()
            pool.read(layer, slots_of(each, at), kv, pe, err)
            q[layer] = (0.3 * torch.cat([kv, pe], 1)[:, None] + 0.3 * rand(requests, heads, d + dr)).bfloat16()

    next_token()
    graphs, ms = {}, {}
    for name in out:
        step(name)  # a first call outside the capture sets the kernels up
        torch.cuda.synchronize()
        graphs[name] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[name]):
            step(name)
        ms[name] = 0.0
    for i in range(steps):
        if i:
            next_token()
        for name, graph in graphs.items():
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            graph.replay()
            end.record()
            torch.cuda.synchronize()
            ms[name] += begin.elapsed_time(end) / steps
    if int(err):
        raise RuntimeError(f"the kernels reported {int(err)}")
    a, c = out["all"].float(), out["chosen"].float()
    # the share of the whole attention's weight that the chosen pages hold
    share = float((lse["chosen"] - lse["all"]).exp().mean())
    return {"ms": ms, "out": out, "lse": lse, "share": share, "error": float((a - c).norm() / a.norm()), "pool": pool, "q": q,
            "table": table, "seq_lens": seq_lens, "sm_scale": sm_scale}


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (("requests", 32), ("context", 32768), ("budget", 32), ("layers", 2), ("steps", 16)):
        p.add_argument(f"--{name}", type=int, default=default)
    a = p.parse_args()
    r = run(a.requests, a.context, a.budget, a.layers, a.steps)
    print(f"{a.requests} requests of {a.context // 2} to {a.context} tokens, {a.layers} layers, cache {r['pool'].get_kv_size_bytes() / 2**20:.0f} MiB")
    print(f"attention over all pages     {r['ms']['all']:.3f} ms a step")
    print(f"over {a.budget:4d} chosen pages      {r['ms']['chosen']:.3f} ms a step, holding {r['share']:.1%} of the weight; "
          f"outputs differ by {r['error']:.2%}")


if __name__ == "__main__":
    main()
