"""One attention layer served with the paged operators: ragged prompts in one
pass, then decode steps over the 4-bit cache.

    python examples/paged_serving.py [--model tinyllama-1.1b] [--requests 8] [--prompt 700] [--decode 32]

A step plans its pages on the device (paged_slots), projects the new tokens
with the framework's int8 ``Linear``, rotates queries and keys by their
positions, appends keys and values to the 4-bit pages and attends: whole
prompts over their own bf16 keys and values, single tokens over the cache.
Nothing but the number of new tokens is known to the host.
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import modelc_b200 as mb  # noqa: E402


class PagedAttention:
    """Projections, rotary table, pool and page tables of one layer."""

    def __init__(self, cfg, requests: int, pages: int, max_context: int, device: int = 0, seed: int = 0,
                 scaling=None):
        self.cfg = cfg
        c = cfg.resolved()
        self.H, self.Hk, self.D = c.n_heads, c.n_kv_heads, c.head_dim
        rng = np.random.default_rng(seed)

        def linear(n_out, n_in):
            w = (rng.standard_normal((n_out, n_in), dtype=np.float32) / np.float32(n_in ** 0.5)).astype(np.float32)
            return mb.Linear(mb.QTensor("i8_row", *mb.quantize_int8_rows(w)), device)

        self.qkv = linear((self.H + 2 * self.Hk) * self.D, c.hidden)
        self.o = linear(c.hidden, self.H * self.D)
        self.cos, self.sin = mb.rope_table(max_context, self.D, c.rope_theta, scaling, device)
        self.pool = mb.kv4_pool(pages, self.Hk, self.D, device)
        dev = self.pool.device
        width = (max_context + mb.paged.PAGE - 1) // mb.paged.PAGE
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device=dev)
        self.free = torch.arange(pages, dtype=torch.int32, device=dev)
        self.n_free = torch.tensor([pages], dtype=torch.int32, device=dev)
        self.kv_len = torch.zeros(requests, dtype=torch.int32, device=dev)

    def step(self, x, q_len, prompts: bool):
        """x [tokens, hidden] (f32): q_len[z] new tokens of each request, one
        behind the other.  ``prompts``: the requests are new and bring their
        whole prompts; otherwise a few tokens each, over the cache.  Returns
        the layer's output [tokens, hidden]."""
        H, Hk, D = self.H, self.Hk, self.D
        plan = mb.paged_slots(self.kv_len, q_len, self.table, self.free, self.n_free, x.shape[0])
        y = self.qkv(x)
        q, k = mb.rope(y[:, :H * D].unflatten(1, (H, D)), y[:, H * D:(H + Hk) * D].unflatten(1, (Hk, D)),
                       plan.positions, self.cos, self.sin, dtype=torch.bfloat16)
        v = y[:, (H + Hk) * D:].unflatten(1, (Hk, D)).to(torch.bfloat16)
        mb.kv4_append(self.pool, k, v, plan.slots)
        if prompts:
            a = mb.prompt_attention(q, k, v, plan.cu_q)
        else:
            a = mb.kv4_attention(q, self.pool, self.table, plan.new_len, plan.cu_q)
        self.kv_len, self.n_free = plan.new_len, plan.n_free
        return x + self.o(a.flatten(1).float())


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--model", default="tinyllama-1.1b", choices=sorted(mb.PRESETS))
    p.add_argument("--requests", type=int, default=8)
    p.add_argument("--prompt", type=int, default=700, help="longest prompt; the others are shorter")
    p.add_argument("--decode", type=int, default=32)
    a = p.parse_args(argv)
    cfg = mb.PRESETS[a.model]
    lens = [max(1, a.prompt * (z + 1) // a.requests) for z in range(a.requests)]
    pages = sum((n + a.decode + 63) // 64 for n in lens)
    layer = PagedAttention(cfg, a.requests, pages, a.prompt + a.decode)
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    x = torch.randn(sum(lens), cfg.hidden, generator=g, device="cuda")
    out = layer.step(x, torch.tensor(lens, dtype=torch.int32, device="cuda"), prompts=True)
    last = out[torch.tensor(lens, device="cuda").cumsum(0) - 1]
    one = torch.ones(a.requests, dtype=torch.int32, device="cuda")
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for i in range(a.decode):
        if i == 1:  # the first step loads the kernels
            start.record()
        last = layer.step(last, one, prompts=False)
        last = last / last.square().mean(1, keepdim=True).sqrt()
    end.record()
    torch.cuda.synchronize()
    took = start.elapsed_time(end) / (a.decode - 1) * 1e3 if a.decode > 1 else 0.0
    print(f"{cfg.name}: {sum(lens)} prompt tokens of {a.requests} requests, then {a.decode} steps of "
          f"{took:.0f} us; {int(layer.n_free)} of {pages} pages left, "
          f"lengths {layer.kv_len.tolist()}")
    return last


if __name__ == "__main__":
    main()
