"""The feed-forward half of a mixture-of-experts decoder layer on 4-bit weights:

    y = x + shared(x) + sum_j weight[j] expert[id[j]](x)

with a shared gated MLP (three W4Linear), a router and routed experts (MoE).  A
prompt of many tokens runs eagerly; single tokens decode from a graph that is
captured once.

    python examples/moe_block.py [--dim 2048 --ffn 1408 --experts 64 --top-k 6]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from hipgemm_amd.torch_serving import MoE, W4Linear  # noqa: E402


class Block(torch.nn.Module):
    def __init__(self, dim, ffn, experts, k, format="int4", group_size=64, seed=0):
        super().__init__()
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*shape):
            w = torch.randn(shape, generator=g, device="cuda") * shape[-1] ** -0.5
            return w.to(torch.bfloat16)

        def linear(n, k_, activation=None):
            lin = torch.nn.Linear(k_, n, bias=False, device="meta")
            lin.weight = torch.nn.Parameter(weight(n, k_), requires_grad=False)
            return W4Linear.from_linear(lin, format, group_size, activation=activation)

        self.gate, self.up = linear(ffn, dim, "silu"), linear(ffn, dim)
        self.down = linear(dim, ffn)
        self.moe = MoE.from_weights(weight(experts, dim), weight(experts, 2 * ffn, dim),
                                    weight(experts, dim, ffn), k, format, group_size)

    def forward(self, x):
        return x + self.down(self.gate(x) * self.up(x)) + self.moe(x)


def capture(block, tokens, dim):
    """(step, x, y): step() decodes x into y; both stay where they are."""
    x = torch.zeros(tokens, dim, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block(x)
    return graph.replay, x, y


def main():
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--dim", type=int, default=2048)
    p.add_argument("--ffn", type=int, default=1408)
    p.add_argument("--experts", type=int, default=64)
    p.add_argument("--top-k", type=int, default=6)
    p.add_argument("--prompt", type=int, default=512)
    p.add_argument("--steps", type=int, default=200)
    a = p.parse_args()
    with torch.no_grad():
        block = Block(a.dim, a.ffn, a.experts, a.top_k)
        prompt = torch.randn(a.prompt, a.dim, device="cuda").to(torch.bfloat16)
        block(prompt)
        torch.cuda.synchronize()
        t = time.perf_counter()
        last = block(prompt)[-1:]
        torch.cuda.synchronize()
        print(f"prompt of {a.prompt} tokens: {(time.perf_counter() - t) * 1e3:.2f} ms")
        step, x, y = capture(block, 1, a.dim)
        x.copy_(last)
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(a.steps):
            step()
        torch.cuda.synchronize()
        print(f"a token: {(time.perf_counter() - t) / a.steps * 1e6:.1f} us, "
              f"of {a.steps} in a graph")
        err = (y - block(x)).abs().max().item()
        print(f"graph against eager: largest difference {err}")


if __name__ == "__main__":
    main()
