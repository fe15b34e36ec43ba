"""A layer of experts with 4-bit weights: the router's scores, its choice, the sorted rows and two products of each expert,
the second summed by weight. ``python -m numkong_amd.examples.experts_layer`` serves a prompt and a few tokens with it, the
latter also from a graph, and trains a router for some steps."""
from __future__ import annotations

import argparse
import time

import torch

import numkong_amd as nk


class ExpertsLayer:
    """``y = sum over the chosen of weight * down[e] @ relu(up[e] @ x)``; activations in bfloat16."""

    def __init__(self, router, up, down, top_k: int, score: str = "softmax", bias=None):
        """``router`` experts x depth in bfloat16, ``up`` experts x hidden x depth, ``down`` experts x depth x hidden."""
        self.router = nk.dots_pack(router, "bf16")
        self.up, self.down = nk.mx_pack(up), nk.mx_pack(down)
        self.top_k, self.score, self.bias = top_k, score, bias

    def scores(self, x):
        """The router's logits, in bfloat16 products: this call waits for its result, and stays out of graphs."""
        return nk.dots_packed(x, self.router)

    def experts(self, x, logits):
        """The layer but for its scores, queued on the current stream."""
        weights, chosen = nk.experts_route(logits, self.top_k, self.score, self.bias)
        plan = nk.experts_plan(chosen, self.up.count)
        hidden = torch.relu(nk.mx_dots_experts(x, self.up, plan, out_dtype=torch.bfloat16))
        return nk.mx_dots_experts(hidden.reshape(-1, self.up.width), self.down, plan, weights, out_dtype=torch.bfloat16)

    def __call__(self, x):
        return self.experts(x, self.scores(x))


def train_router(x, wanted, experts: int, top_k: int, steps: int, rate: float = 0.5):
    """Teaches a router to give the weight of each token to its `wanted` expert; (first loss, last loss)."""
    router = torch.zeros((x.shape[1], experts), device=x.device, requires_grad=True)
    losses = []
    for _ in range(steps):
        logits = x @ router
        weights, chosen = nk.experts_route(logits, top_k)  # (weights have a gradient)
        hit = chosen == wanted[:, None]
        # a token whose expert is not among the chosen pulls it up through the scores of all
        loss = ((1 - (weights * hit).sum(1)) * hit.any(1)).mean() + torch.nn.functional.cross_entropy(logits, wanted) * 0.5
        router.grad = None
        loss.backward()
        with torch.no_grad():
            router -= rate * router.grad
        losses.append(loss.detach())
    return float(losses[0]), float(losses[-1])


def make(experts: int, hidden: int, depth: int, top_k: int, seed: int = 0, device: str = "cuda:0"):
    """A layer of random weights and the weights themselves."""
    generator = torch.Generator(device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device=device, dtype=torch.bfloat16, generator=generator) / shape[-1] ** 0.5

    router, up, down = normal(experts, depth) * depth**0.5 / 4, normal(experts, hidden, depth), normal(experts, depth, hidden)
    return ExpertsLayer(router, up, down, top_k), (router, up, down)


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--experts", type=int, default=64)
    parser.add_argument("--top-k", type=int, default=8)
    parser.add_argument("--hidden", type=int, default=2048)
    parser.add_argument("--depth", type=int, default=2048)
    parser.add_argument("--prompt", type=int, default=4096)
    options = parser.parse_args(argv)
    layer, _ = make(options.experts, options.hidden, options.depth, options.top_k)

    def normal(tokens):
        return torch.randn((tokens, options.depth), device="cuda:0", dtype=torch.bfloat16)

    def milliseconds(step, repeats=20):
        step()
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(repeats):
            step()
        torch.cuda.synchronize()
        return (time.perf_counter() - start) / repeats * 1e3

    prompt, token = normal(options.prompt), normal(4)
    print(f"prompt of {options.prompt}: {milliseconds(lambda: layer(prompt)):.3f} ms")
    print(f"4 tokens: {milliseconds(lambda: layer(token)):.3f} ms")
    logits = layer.scores(token)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.experts(token, logits)
    print(f"4 tokens, all but the scores from a graph: {milliseconds(graph.replay):.3f} ms, the same values: {bool((y == layer(token)).all())}")
    wanted = torch.randint(0, options.experts, (1024,), device="cuda:0")
    x = torch.nn.functional.one_hot(wanted, options.depth).float() + 0.1 * torch.randn((1024, options.depth), device="cuda:0")
    print("loss of the router: %.3f -> %.3f" % train_router(x, wanted, options.experts, options.top_k, 50, 20.0))


if __name__ == "__main__":
    main()
