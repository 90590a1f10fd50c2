"""Trains the feed-forward half of a decoder layer in 16 bits and decodes with it:

    y = x + down(silu(gate(x)) * up(x))

GatedMLP is two calls forward (gated_linear, then linear with the residual in its
epilogue) and two backward.  The target is another block's output.  After the training the
weights serve single tokens from a captured graph, or are quantised (--w4) to W4Linear.

    python examples/train_block.py [--dim 1024 --hidden 2816 --tokens 2048 --steps 50]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from hipgemm_amd.torch_dense import GatedMLP  # noqa: E402
from hipgemm_amd.torch_serving import W4Linear  # noqa: E402


def make(dim, hidden, seed):
    torch.manual_seed(seed)
    return GatedMLP(dim, hidden, device="cuda")


def gradients(block, x, target):
    """(loss, gradients of w13 and w2) of the mean squared error."""
    y = block(x, residual=x)
    loss = (y.float() - target.float()).square().mean()
    return loss.detach(), torch.autograd.grad(loss, (block.w13, block.w2))


def train(block, x, target, steps, rate=1e-3):
    """Adam on float32 copies of the weights; returns the losses."""
    master = [p.detach().float() for p in (block.w13, block.w2)]
    opt = torch.optim.Adam(master, lr=rate)
    losses = []
    for _ in range(steps):
        loss, grads = gradients(block, x, target)
        for m, g in zip(master, grads):
            m.grad = g.float()
        opt.step()
        with torch.no_grad():
            for p, m in zip((block.w13, block.w2), master):
                p.copy_(m)
        losses.append(loss)
    return losses


def capture(block, dim):
    """(step, x, y): step() runs the block on x into y, which stay where they are."""
    x = torch.zeros(1, dim, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        block(x, residual=x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = block(x, residual=x)
    return graph.replay, x, y


def main():
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--dim", type=int, default=1024)
    p.add_argument("--hidden", type=int, default=2816)
    p.add_argument("--tokens", type=int, default=2048)
    p.add_argument("--steps", type=int, default=50)
    p.add_argument("--w4", action="store_true", help="also quantise the trained weights")
    a = p.parse_args()
    block, goal = make(a.dim, a.hidden, 0), make(a.dim, a.hidden, 1)
    x = torch.randn(a.tokens, a.dim, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        target = goal(x, residual=x)
    train(block, x, target, 2)
    torch.cuda.synchronize()
    t = time.perf_counter()
    losses = train(block, x, target, a.steps)
    torch.cuda.synchronize()
    print(f"a step of {a.tokens} tokens: {(time.perf_counter() - t) / a.steps * 1e3:.3f} ms; "
          f"loss {losses[0].item():.4f} -> {losses[-1].item():.4f}")
    step, sx, sy = capture(block, a.dim)
    sx.copy_(x[:1])
    for _ in range(3):
        step()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(200):
        step()
    torch.cuda.synchronize()
    print(f"a token: {(time.perf_counter() - t) / 200 * 1e6:.1f} us in a graph")
    with torch.no_grad():
        print(f"graph against eager: largest difference "
              f"{(sy - block(x[:1], residual=x[:1])).abs().max().item()}")
        if a.w4:
            def linear(w, activation=None):
                lin = torch.nn.Linear(w.shape[1], w.shape[0], bias=False, device="meta")
                lin.weight = torch.nn.Parameter(w, requires_grad=False)
                return W4Linear.from_linear(lin, "int4", 64, activation=activation)
            gate, up = block.w13.detach().chunk(2)
            h = linear(gate, "silu")(x) * linear(up)(x)
            y = x + linear(block.w2.detach())(h)
            err = (y.float() - block(x, residual=x).float()).square().mean().sqrt()
            print(f"int4 weights: rms difference {err.item():.4f}")


if __name__ == "__main__":
    main()
