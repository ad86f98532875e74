"""A layer of a small random language model over the paged 4-bit cache: prompts of different lengths, then decode steps.

    python examples/paged_step.py [--requests 4] [--steps 8]

Each step is what a server runs: the block tables and slot maps on the GPU (paged.plan), then for the layer the fused 4-bit
QKV projection, the cache write with rotary positions (paged.append), attention over the pages (paged.attend) and the 4-bit
output projection. Prints the tokens in the cache and the time a step takes.
"""

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from locals_b200 import kernels, paged, rotary
from locals_b200.fuse import FusedQKV
from locals_b200.kernels import QuantizedLinear


def projection(rows, cols, gen, device):
    w = torch.randn((rows, cols), generator=gen, device=device) * 0.02
    return QuantizedLinear(*kernels.quantize(w.to(torch.bfloat16), bits=4))


class Layer:
    """Attention of one layer: hidden 2560, 32 query heads on 8 key/value heads of 128."""

    def __init__(self, pages, page, gen, device, hidden=2560, heads=32, kv_heads=8, dim=128):
        self.scale = dim ** -0.5
        q, k, v = (projection(h * dim, hidden, gen, device) for h in (heads, kv_heads, kv_heads))
        self.qkv = FusedQKV(q, k, v, heads, kv_heads, dim)
        self.out = projection(hidden, heads * dim, gen, device)
        self.keys, self.values = paged.pool(pages, kv_heads, page, dim, torch.bfloat16, device)

    def __call__(self, x, p, table, max_q, cos, sin):
        q, k, v = self.qkv(x)
        q = paged.append(q, k, v, p.slots, self.keys, self.values, p.positions, cos, sin)
        o = paged.attend(q, self.keys, self.values, table, p.lens, self.scale, q_start=p.q_start, max_q=max_q)
        return self.out(o.reshape(len(x), -1))


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args(argv)
    dev, page, longest = torch.device("cuda"), 16, 512
    gen = torch.Generator(device=dev)
    gen.manual_seed(0)
    width = (longest + a.steps + page - 1) // page
    layer = Layer(a.requests * width, page, gen, dev)
    cos, sin = rotary.tables(longest + a.steps, 128, device=dev)
    table = torch.full((a.requests, width), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(a.requests * width, generator=gen, device=dev).to(torch.int32)
    head, cached = torch.zeros(1, dtype=torch.int32, device=dev), torch.zeros(a.requests, dtype=torch.int32, device=dev)
    prompts = [longest - 37 * b % longest for b in range(a.requests)]
    for step in range(a.steps + 1):
        new = prompts if step == 0 else [1] * a.requests
        x = torch.randn((sum(new), 2560), generator=gen, device=dev).to(torch.bfloat16)
        fresh = torch.tensor(new, dtype=torch.int32, device=dev)
        torch.cuda.synchronize()
        t = time.perf_counter()
        p = paged.plan(cached, fresh, table, free, head, page, sum(new))
        y = layer(x, p, table, max(new), cos, sin)
        torch.cuda.synchronize()
        print(f"step {step}: {sum(new)} new tokens, {int(p.lens.sum())} cached in {int(p.head)} pages, "
              f"{(time.perf_counter() - t) * 1e6:.0f} us, |y| {float(y.float().abs().mean()):.4f}")
        assert bool(torch.isfinite(y).all()) and kernels.device_status() == 0
        cached, head = p.lens, p.head


if __name__ == "__main__":
    main()
