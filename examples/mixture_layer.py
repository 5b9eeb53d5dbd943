"""A mixture-of-experts layer in MXFP4, as a server runs it: fp32 weights are quantised once, then every step multiplies the tokens by the
router, chooses experts, runs their gated feed-forward, and adds a dense feed-forward's output projection beside it.

    python examples/mixture_layer.py [--tokens 1,64,2048] [--hidden 2048] [--expert 512] [--experts 32] [--top 4]

Weights are random; prints how far the layer's output is from one in fp32 with unrounded weights, and the time of a step replayed from a graph.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import ruquant_amd as rq  # noqa: E402


class MixtureLayer:
    def __init__(self, hidden, expert, experts, top, device="cuda:0", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        random = lambda *shape: torch.randn(shape, device=device, generator=g) * shape[-1] ** -0.5  # noqa: E731
        self.top = top
        self.fp32 = {"router": random(experts, hidden), "gate": random(experts, expert, hidden), "up": random(experts, expert, hidden),
                     "down": random(experts, hidden, expert), "shared": random(hidden, hidden)}
        self.bias = 0.02 * torch.randn((experts,), device=device, generator=g)
        self.weights = {name: self.quantise(w) for name, w in self.fp32.items()}

    @staticmethod
    def quantise(w):
        codes, scales = rq.mx_quantize(w.flatten(0, -2))
        return rq.MXWeight(codes.view(*w.shape[:-1], -1), scales.view(*w.shape[:-1], -1))

    def __call__(self, x):
        w = self.weights
        logits = rq.mx_mul_mat(w["router"], x, out=x.new_empty((x.shape[0], w["router"].N), dtype=torch.float32))
        ids, share = rq.route(logits, self.top, scoring="sigmoid", bias=self.bias)
        return rq.expert_ffn(w["gate"], w["up"], w["down"], x, ids, share) + rq.mx_mul_mat(w["shared"], x), ids, share

    def in_fp32(self, x, ids, share):
        """the same experts and shares, nothing rounded"""
        w, x = self.fp32, x.float()
        y = x @ w["shared"].t()
        for e in range(w["gate"].shape[0]):
            t, j = (ids == e).nonzero(as_tuple=True)
            if len(t):
                h = torch.nn.functional.silu(x[t] @ w["gate"][e].t()) * (x[t] @ w["up"][e].t())
                y.index_add_(0, t, share[t, j, None] * (h @ w["down"][e].t()))
        return y


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--tokens", default="1,64,2048")
    p.add_argument("--hidden", type=int, default=2048)
    p.add_argument("--expert", type=int, default=512)
    p.add_argument("--experts", type=int, default=32)
    p.add_argument("--top", type=int, default=4)
    a = p.parse_args(argv)
    layer = MixtureLayer(a.hidden, a.expert, a.experts, a.top)
    off = []
    for tokens in map(int, a.tokens.split(",")):
        x = torch.randn((tokens, a.hidden), device="cuda:0").bfloat16()
        y, ids, share = layer(x)
        want = layer.in_fp32(x, ids, share)
        off.append(((y.float() - want).norm() / want.norm()).item())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer(x)
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        graph.replay()
        begin.record()
        for _ in range(20):
            graph.replay()
        end.record()
        torch.cuda.synchronize()
        print("%5d tokens: %7.1f us a step, %.3f off fp32" % (tokens, begin.elapsed_time(end) / 20 * 1e3, off[-1]))
    return off


if __name__ == "__main__":
    main()
