"""The workspace of attention over the 4-bit cache: nothing of it stays behind
a call, and calls that run side by side do not share one."""
import gc
import threading

import pytest

import modelc_b200 as mb

gpu = pytest.mark.gpu


def _case(requests, H, Hk, D, n, seed):
    """Arguments of a call of one token each, over one shared context."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    pages = (n + 63) // 64
    pool = mb.kv4_pool(pages, Hk, D)
    mb.kv4_append(pool, randn(n, Hk, D), randn(n, Hk, D), torch.arange(n, dtype=torch.int32, device="cuda"))
    return (randn(requests, H, D).bfloat16(), pool,
            torch.arange(pages, dtype=torch.int32, device="cuda").repeat(requests, 1),
            torch.full((requests,), n, dtype=torch.int32, device="cuda"),
            torch.arange(requests + 1, dtype=torch.int32, device="cuda"))


@gpu
def test_nothing_is_kept():
    """Streams and threads come and go; the memory in use is what it was."""
    import torch
    args = _case(3, 8, 2, 128, 500, 1)
    want = mb.kv4_attention(*args)
    gc.collect()  # what earlier tests left in cycles
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before, reserved = torch.cuda.memory_allocated(), torch.cuda.memory_reserved()
    seen = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            seen.append(torch.equal(mb.kv4_attention(*args), want))
        torch.cuda.synchronize()

    for _ in range(4):
        work()
    threads = [threading.Thread(target=work) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert seen == [True] * 10
    assert torch.cuda.memory_allocated() == before
    torch.cuda.empty_cache()
    assert torch.cuda.memory_reserved() <= reserved + (20 << 20)  # one workspace is 19 MB


@gpu
def test_sizes_that_grow_and_shrink():
    """Calls of different sizes after one another on one stream."""
    import torch
    cases = [_case(1, 8, 2, 64, 300, 2), _case(700, 8, 2, 64, 300, 3), _case(2, 8, 2, 128, 3000, 4),
             _case(900, 4, 4, 128, 100, 5)]
    want = [mb.kv4_attention(*c) for c in cases]
    torch.cuda.synchronize()
    for order in ((0, 1, 2, 3), (3, 2, 1, 0), (1, 0, 3, 0, 2)):
        got = [(i, mb.kv4_attention(*cases[i])) for i in order]
        assert all(torch.equal(x, want[i]) for i, x in got)


@gpu
def test_threads_on_one_stream():
    """Two threads' calls alternate on one stream."""
    import torch
    cases = [_case(2, 8, 2, 128, 4000, 6), _case(5, 8, 2, 128, 2500, 7)]
    want = [mb.kv4_attention(*c) for c in cases]
    torch.cuda.synchronize()
    stream, good = torch.cuda.Stream(), [0, 0]

    def work(i):
        for _ in range(40):
            with torch.cuda.stream(stream):
                good[i] += torch.equal(mb.kv4_attention(*cases[i]), want[i])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert good == [40, 40]
