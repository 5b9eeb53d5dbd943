"""A layer of experts in 8-bit integers or in 16 bits, as a server runs it on the products grouped by expert: the router's choices are sorted by expert, gate
and up projections read the tokens where they lie, the activation between is the caller's own, the down projection writes to the slots' places, and a token's slots are added up.

    python examples/int8_experts.py [--weights int8|bf16] [--tokens 1,64,2048] [--hidden 2048] [--expert 512] [--experts 32] [--top 4]

Weights are random; prints how far the layer's output is from one in fp32 with unrounded weights, and the time of a step replayed from a graph.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import ruquant_amd as rq  # noqa: E402


class ExpertsLayer:
    def __init__(self, hidden, expert, experts, top, weights="int8", device="cuda:0", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        random = lambda *shape: torch.randn(shape, device=device, generator=g) * shape[-1] ** -0.5  # noqa: E731
        self.top, self.experts = top, experts
        self.router = random(experts, hidden).bfloat16()
        self.fp32 = {"gate": random(experts, expert, hidden), "up": random(experts, expert, hidden), "down": random(experts, hidden, expert)}
        self.weights = {name: self.int8(w) if weights == "int8" else rq.HalfWeight(w.bfloat16()) for name, w in self.fp32.items()}

    @staticmethod
    def int8(w):
        codes, scales = rq.i8_quantize(w.flatten(0, -2))
        return rq.I8Weight(codes.view(w.shape), scales.view(w.shape[:-1]))

    def __call__(self, x):
        w = self.weights
        ids, share = rq.route(x @ self.router.t(), self.top)
        offsets, slots, tokens = rq.sort_slots(ids, self.experts)
        if isinstance(w["gate"], rq.I8Weight):   # rounded once for both
            rows, scales = rq.i8_quantize(x)
        else:
            rows, scales = x, None
        gate, up = (rq.grouped_mul_mat(w[name], rows, offsets, rows=tokens, scales=scales, dtype=x.dtype) for name in ("gate", "up"))
        h = torch.nn.functional.silu(gate) * up
        y = rq.grouped_mul_mat(w["down"], h, offsets, out_rows=slots, dtype=torch.float32)
        return (y.view(*ids.shape, -1) * share[:, :, None]).sum(dim=1).to(x.dtype), ids, share

    def in_fp32(self, x, ids, share):
        """the same experts and shares, nothing rounded"""
        w, x = self.fp32, x.float()
        y = torch.zeros_like(x)
        for e in range(self.experts):
            t, j = (ids == e).nonzero(as_tuple=True)
            if len(t):
                h = torch.nn.functional.silu(x[t] @ w["gate"][e].t()) * (x[t] @ w["up"][e].t())
                y.index_add_(0, t, share[t, j, None] * (h @ w["down"][e].t()))
        return y


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--weights", choices=("int8", "bf16"), default="int8")
    p.add_argument("--tokens", default="1,64,2048")
    p.add_argument("--hidden", type=int, default=2048)
    p.add_argument("--expert", type=int, default=512)
    p.add_argument("--experts", type=int, default=32)
    p.add_argument("--top", type=int, default=4)
    a = p.parse_args(argv)
    layer = ExpertsLayer(a.hidden, a.expert, a.experts, a.top, a.weights)
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
        print("%5d tokens: %7.1f us a step, %.4f off fp32" % (tokens, begin.elapsed_time(end) / 20 * 1e3, off[-1]))
    return off


if __name__ == "__main__":
    main()
