"""The feed-forward part of a decoder layer with 8-bit floating-point weights: norm, router, experts and the shared expert.

    python examples/expert_layer.py [--tokens 64] [--steps 4] [--dtype bf16|f16|f32] [--graph]

Weights are e4m3 with a scale for each block of 128 x 128 and random.  Each step normalises the tokens into 8 bits, sorts
them by expert, runs the experts' gate, up and down products and the shared expert's, and adds the rows up; with --graph the
step is captured once and replayed on new tokens.  The last step is recomputed in 64 bits without the two 8-bit roundings on
the way, and the relative error is printed (and returned by `main`).
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from dracomancer_llmengine_b200 import decoder  # noqa: E402

HIDDEN, EXPERTS, USED, INTER, SHARED, EPS = 2048, 32, 4, 512, 512, 1e-6
E4M3 = torch.float8_e4m3fn


def quantise(w):
    """e4m3 codes and 128 x 128 block scales of weights [..., n, k] (n and k multiples of 128)."""
    blocks = w.unflatten(-1, (-1, 128)).unflatten(-3, (-1, 128))                # [..., n/128, 128, k/128, 128]
    scales = blocks.abs().amax((-3, -1)) / 448
    return (blocks / scales[..., :, None, :, None]).to(E4M3).flatten(-2).flatten(-3, -2).contiguous(), scales.contiguous()


def values(codes, scales):
    """Weights in 64 bits."""
    return codes.double() * scales.double().repeat_interleave(128, -2).repeat_interleave(128, -1)


class Layer:
    """Weights of one layer, and the buffers of a step of `tokens` tokens."""

    def __init__(self, tokens, dtype, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        make = lambda *s: torch.randn(*s, device="cuda", generator=gen) / s[-1] ** 0.5  # noqa: E731
        self.router, self.norm = make(EXPERTS, HIDDEN), 1 + 0.1 * torch.randn(HIDDEN, device="cuda", generator=gen)
        self.gate_up, self.down = quantise(make(EXPERTS, 2, INTER, HIDDEN)), quantise(make(EXPERTS, HIDDEN, INTER))
        self.shared_gate_up, self.shared_down = quantise(make(2, SHARED, HIDDEN)), quantise(make(HIDDEN, SHARED))
        empty = lambda *s, t=torch.float32: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731
        self.x, self.y, self.out = (torch.zeros(tokens, HIDDEN, dtype=dtype, device="cuda") for _ in range(3))
        self.rows = (empty(tokens, HIDDEN, t=E4M3), empty(tokens, HIDDEN // 128))
        self.plan = decoder.ExpertPlan(tokens, USED, EXPERTS)
        self.act = (empty(tokens * USED, INTER, t=E4M3), empty(tokens * USED, INTER // 128))
        self.shared_act = (empty(tokens, SHARED, t=E4M3), empty(tokens, SHARED // 128))
        self.expert_rows, self.shared = empty(tokens * USED, HIDDEN, t=dtype), empty(tokens, HIDDEN, t=dtype)

    def step(self):
        """out = the layer's feed-forward of x."""
        decoder.rmsnorm_q8(self.x, self.norm, EPS, *self.rows, y=self.y, group=128)
        score, chosen = (self.y.float() @ self.router.T).softmax(-1).topk(USED, -1)
        self.chosen, self.weights = chosen.int(), score / score.sum(-1, keepdim=True)
        plan = decoder.plan_experts(self.chosen, self.plan)
        decoder.swiglu_q8(*self.rows, *self.gate_up, *self.act, offsets=plan.offsets, rows=plan.rows)
        decoder.linear_q8(*self.act, *self.down, self.expert_rows, offsets=plan.offsets)
        decoder.swiglu_q8(*self.rows, *self.shared_gate_up, *self.shared_act)
        decoder.linear_q8(*self.shared_act, *self.shared_down, self.shared)
        decoder.combine_experts(self.expert_rows, plan.pos, self.weights, self.out, add=self.shared)

    def error(self):
        """Relative error of the last step against 64 bits over the weights' own values and the step's own routing."""
        x = self.x.double()
        h = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * self.norm.double()

        def ffn(rows, gate_up, down):
            g, u = rows @ gate_up[0].T, rows @ gate_up[1].T
            return (g * torch.sigmoid(g) * u) @ down.T

        want = ffn(h, values(*self.shared_gate_up), values(*self.shared_down))
        for e in range(EXPERTS):
            t, k = (self.chosen == e).nonzero(as_tuple=True)
            if len(t):
                y = ffn(h[t], *(values(c[e], s[e]) for c, s in (self.gate_up, self.down)))
                want.index_add_(0, t, y * self.weights[t, k, None].double())
        return float(torch.linalg.norm(self.out.double() - want) / torch.linalg.norm(want))


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--steps", type=int, default=4)
    ap.add_argument("--dtype", choices=("bf16", "f16", "f32"), default="bf16")
    ap.add_argument("--graph", action="store_true")
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    layer = Layer(a.tokens, {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[a.dtype])
    step = layer.step
    if a.graph:
        step()                                  # the libraries behind the router set themselves up outside of the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer.step()
        step = graph.replay
    for _ in range(a.steps):
        layer.x.copy_(torch.randn(layer.x.shape, device="cuda"))
        step()
    error = layer.error()
    print(f"{a.steps} steps of {a.tokens} tokens, {EXPERTS} experts of {INTER}, {USED} a token: relative error {error:.1e}")
    return error


if __name__ == "__main__":
    main()
