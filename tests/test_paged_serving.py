"""The paged operators together, as examples/paged_serving.py runs them."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hk,d", [(4, 64), (2, 128)])
def test_steps_agree_with_the_tokens_one_by_one(hk, d):
    """Prompts in one pass, then a step of several tokens, against the layer's
    definition in 64 bits over the values that the cache holds.

    Tolerance: rotated queries and attention outputs are rounded to bf16
    (2^-8 each) and weights to f16 (2^-11, twice); the output projection sums
    H D of these errors with random signs at weights of variance 1 / (H D),
    so 2^-6 of an output of size 1 leaves a factor of four."""
    import torch
    import modelc_b200 as mb
    import paged_serving as ps
    cfg = mb.LlamaConfig(1, 256, 8, hk, d, 512, 100, 10000.0)
    layer = ps.PagedAttention(cfg, 3, 20, 400)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    lens, news = [130, 1, 64], [2, 3, 1]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    x = torch.randn(sum(lens), 256, generator=g, device="cuda")
    layer.step(x, t(lens), True)
    assert layer.kv_len.tolist() == lens and int(layer.n_free) == 20 - 3 - 1 - 1
    y = torch.randn(sum(news), 256, generator=g, device="cuda")
    out = layer.step(y, t(news), False)
    assert layer.kv_len.tolist() == [132, 4, 65] and int(layer.n_free) == 20 - 3 - 1 - 2
    f, _ = mb.rope_frequencies(d, 10000.0)
    f = torch.tensor(f, device="cuda", dtype=torch.float64)
    a = 0
    for z, (n, m) in enumerate(zip(lens, news)):
        L = n + m
        j = torch.arange(L, device="cuda")
        slots = (layer.table[z, j // 64] * 64 + j % 64).to(torch.int32)
        k, v = (c.double().repeat_interleave(8 // hk, 1) for c in mb.kv4_read(layer.pool, slots, d, torch.float32))
        q = layer.qkv(y[a:a + m])[:, :8 * d].double().view(m, 8, 2, d // 2)
        at = torch.arange(n, L, device="cuda").double()[:, None, None] * f
        q = torch.cat([q[:, :, 0] * at.cos() - q[:, :, 1] * at.sin(), q[:, :, 1] * at.cos() + q[:, :, 0] * at.sin()], -1)
        s = torch.einsum("nhd,lhd->hnl", q, k) / d ** 0.5
        s = s.masked_fill(j > torch.arange(n, L, device="cuda")[:, None], -float("inf"))
        ref = torch.einsum("hnl,lhd->nhd", s.softmax(-1), v).reshape(m, -1)
        ref = y[a:a + m].double() + layer.o(ref.float()).double()
        assert (out[a:a + m].double() - ref).abs().max() <= 2.0 ** -6
        a += m


def test_example_runs():
    import paged_serving as ps
    last = ps.main(["--model", "tiny-4L-d256", "--requests", "3", "--prompt", "100", "--decode", "4"])
    assert last.isfinite().all() and last.shape == (3, 256)


def test_step_in_a_graph():
    """A decode step captured once and replayed gives the step's results."""
    import torch
    import modelc_b200 as mb
    import paged_serving as ps
    cfg = mb.LlamaConfig(1, 256, 4, 4, 64, 512, 100, 10000.0)
    layer = ps.PagedAttention(cfg, 2, 10, 300)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    layer.step(torch.randn(70, 256, device="cuda"), t([50, 20]), True)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    k, v = torch.randn(2, 2, 4, 64, device="cuda").bfloat16()
    one, pos0 = t([1, 1]), layer.kv_len.clone()

    def step():
        plan = mb.paged_slots(pos0, one, layer.table, layer.free, layer.n_free, 2)
        rq, rk = mb.rope(q, k, plan.positions, layer.cos, layer.sin)
        mb.kv4_append(layer.pool, rk, v, plan.slots)
        return mb.kv4_attention(rq, layer.pool, layer.table, plan.new_len, plan.cu_q)

    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, step()) and not torch.equal(got, want)


def test_other_streams():
    """Calls on a stream of their own, two at a time on two streams."""
    import torch
    import modelc_b200 as mb
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    pool = mb.kv4_pool(64, 2, 128)
    k, v = torch.randn(2, 3000, 2, 128, generator=g, device="cuda")
    slots = torch.arange(3000, dtype=torch.int32, device="cuda")
    mb.kv4_append(pool, k, v, slots)
    table = torch.arange(47, dtype=torch.int32, device="cuda")[None]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q = [torch.randn(1, 16, 128, generator=g, device="cuda").half() for _ in range(8)]
    args = (pool, table, t([3000]), t([0, 1]))
    want = [mb.kv4_attention(x, *args) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, x in enumerate(q):
        with torch.cuda.stream(streams[i % 2]):
            got.append(mb.kv4_attention(x, *args))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
