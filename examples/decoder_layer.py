"""One decoder layer served on the GPU: ragged prompts in chunks, then single tokens, for several requests at once.

    python examples/decoder_layer.py [--requests 6] [--steps 8] [--dtype bf16|f16|f32] [--window 0] [--sinks 0]

Each step gives the requests pages for their new tokens, normalises (with the residual's addition), projects, writes keys
and values into the 4-bit cache, attends to it, and runs the quantised mixture-of-experts FFN.  Weights and tokens are
random; rotary positions are left out.  At the end the last step's attention is recomputed in 64 bits from the cache's own
values, and the relative error is printed (and returned by `main`).
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import dracomancer_llmengine_b200 as dm  # noqa: E402
from dracomancer_llmengine_b200 import decoder, synth  # noqa: E402

HEADS, KV_HEADS, DIM, PAGE, EPS = 16, 2, 128, 32, 1e-6


class Layer:
    """Projections (plain matrix products), norms and the MoE FFN of one layer."""

    def __init__(self, dtype, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        make = lambda *s: (torch.randn(*s, device="cuda", generator=gen) / s[0] ** 0.5).to(dtype)  # noqa: E731
        self.moe = synth.make_layer(hidden=2048, n_exp=32, n_used=4, inter=512, shared_inter=512, seed=seed)
        self.hidden, self.dtype = self.moe.hidden, dtype
        self.qkv, self.out = make(self.hidden, (HEADS + 2 * KV_HEADS) * DIM), make(HEADS * DIM, self.hidden)
        self.norm_attn = 1 + 0.1 * torch.randn(self.hidden, device="cuda", generator=gen)
        self.norm_ffn = 1 + 0.1 * torch.randn(self.hidden, device="cuda", generator=gen)


class Server:
    """The requests' state on the GPU: lengths, block table, free pages, the cache."""

    def __init__(self, layer, requests, max_len, window=0, sinks=0):
        per = -(-max_len // PAGE)
        self.layer, self.max_len, self.window, self.sinks = layer, max_len, window, sinks
        self.cache = decoder.KV4Cache.empty(requests * per + 1, PAGE, KV_HEADS, DIM)
        ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.ctx, self.n_free = torch.zeros(requests, dtype=torch.int32, device="cuda"), ints(requests * per)
        self.free = torch.randperm(requests * per, device="cuda").int()
        self.table = torch.full((requests, per), -1, dtype=torch.int32, device="cuda")

    def step(self, x, residual, new_len, max_new):
        """Run the layer on x [tokens, hidden]: new_len[r] tokens of each request, at most max_new."""
        lay, n = self.layer, x.shape[0]
        plan = decoder.BlockPlan(len(new_len), n)
        decoder.plan_blocks(self.ctx, new_len, self.table, self.free, self.n_free, PAGE, plan)
        codes = torch.empty(n, lay.hidden, dtype=torch.int8, device="cuda")   # for consumers that take 8-bit rows
        scales = torch.empty(n, lay.hidden // 256, device="cuda")
        y = torch.empty_like(x)
        decoder.rmsnorm_q8(x, lay.norm_attn, EPS, codes, scales, residual=residual, h=residual, y=y, group=256)
        qkv = (y @ lay.qkv).view(n, HEADS + 2 * KV_HEADS, DIM)
        q, k, v = qkv.split((HEADS, KV_HEADS, KV_HEADS), 1)
        self.cache.append(k, v, plan.slots)
        attended = torch.empty(n, HEADS, DIM, dtype=x.dtype, device="cuda")
        self.cache.attend(q, attended, plan.cu_new, plan.seq_len, self.table, max_new, self.max_len, window=self.window,
                          sinks=self.sinks)
        self.ctx, self.n_free = plan.seq_len, plan.n_free
        x = attended.view(n, -1) @ lay.out
        decoder.rmsnorm_q8(x, lay.norm_ffn, EPS, codes, scales, residual=residual, h=residual, y=y, group=256)
        ffn = torch.empty(n, lay.hidden, device="cuda")
        dm.forward(lay.moe, y.float(), out=ffn, stream=torch.cuda.current_stream())
        self.last = (q, attended, plan)
        return ffn.to(x.dtype)

    def check(self):
        """Relative error of the last step's attention against 64 bits, over the cache's own values.  Raises where the step
        had no pages for a request."""
        q, got, plan = self.last
        if int(plan.refused):       # read with the results: rows of requests without pages mean nothing
            raise RuntimeError(f"{int(plan.refused)} requests found no free page in this step")
        want = torch.zeros(got.shape, dtype=torch.float64, device="cuda")
        cu, seq = plan.cu_new.tolist(), plan.seq_len.tolist()
        for r, n in enumerate(seq):
            pos = torch.arange(n, device="cuda")
            slots = self.table[r, pos // PAGE] * PAGE + (pos % PAGE).int()
            k = torch.empty(n, KV_HEADS, DIM, device="cuda")
            k, v = self.cache.read(slots, k, torch.empty_like(k))
            k, v = (t.double().repeat_interleave(HEADS // KV_HEADS, 1) for t in (k, v))
            at = torch.arange(n - (cu[r + 1] - cu[r]), n, device="cuda")[:, None]
            hidden = pos > at
            if self.window:
                hidden |= (pos <= at - self.window) & (pos >= self.sinks)
            s = torch.einsum("qhd,khd->hqk", q[cu[r]:cu[r + 1]].double(), k) * DIM ** -0.5
            p = s.masked_fill(hidden, -torch.inf).softmax(-1)
            want[cu[r]:cu[r + 1]] = torch.einsum("hqk,khd->qhd", p, v)
        return float(torch.linalg.norm(got.double() - want) / torch.linalg.norm(want))


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--dtype", choices=("bf16", "f16", "f32"), default="bf16")
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    a = ap.parse_args(argv)
    dtype = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[a.dtype]
    torch.manual_seed(0)
    layer = Layer(dtype)
    prompts = [37 + 61 * r for r in range(a.requests)]
    server = Server(layer, a.requests, max(prompts) + a.steps, a.window, a.sinks)
    errors = []
    for chunk in [[-(-p // 2) for p in prompts], [p // 2 for p in prompts]] + [[1] * a.requests] * a.steps:
        x = torch.randn(sum(chunk), layer.hidden, device="cuda").to(dtype)
        server.step(x, torch.randn_like(x), torch.tensor(chunk, dtype=torch.int32, device="cuda"), max(chunk))
        errors.append(server.check())
    print(f"{a.requests} requests, {a.steps} decode steps after prompts of {prompts[0]}..{prompts[-1]} tokens: "
          f"{int(server.ctx.sum())} tokens cached, {int(server.n_free)} pages free, largest error {max(errors):.1e}")
    return errors


if __name__ == "__main__":
    main()
