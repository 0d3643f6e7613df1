"""Attention of the paged operators over the range that values and weights have
in models: small values, and rows most of whose mass one key takes.

Tolerance.  A row's second product rounds every weight times scale, p d, by
itself: f16 over the 4-bit cache (bf16 calls round p and p d), the inputs' type
over prompts.  A rounding of unit roundoff u has a root mean square below u, so
sums of independent ones have one below u sqrt(sum p^2 v^2); the output's own
rounding and the f32 part (2^-12 |o|) come on top, and f16 outputs have steps of
2^-24 near 0.  The root mean square of the error over at least a thousand
outputs has to stay within twice the root mean square of that, which leaves no
room for weights that lose bits, or vanish, for being small.
"""
import math

import pytest

import modelc_b200 as mb

gpu = pytest.mark.gpu
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _rms(x):
    return float(x.double().square().mean().sqrt())


def _exact(q, k, v, see, scale):
    """o and sqrt(sum p^2 v^2) of q [n, H, D] over k, v [L, Hk, D] in 64 bits; row i sees see[i] keys."""
    import torch
    G = q.shape[1] // k.shape[1]
    out, var = torch.empty_like(q, dtype=torch.float64), torch.empty_like(q, dtype=torch.float64)
    hidden = torch.arange(k.shape[0], device=q.device) >= see[:, None]
    for h in range(q.shape[1]):
        kh, vh = k[:, h // G].double(), v[:, h // G].double()
        for r in range(0, q.shape[0], 256):
            x = q[r:r + 256, h].double() @ kh.T * scale
            p = x.masked_fill(hidden[r:r + 256], -math.inf).softmax(-1)
            out[r:r + 256, h], var[r:r + 256, h] = p @ vh, (p * p) @ (vh * vh)
    return out, var.sqrt()


def _inputs(n, rows, H, Hk, D, size, mass, seed):
    """Queries whose scores with n keys are about standard normal, but for key
    0, which takes the share `mass` of a row (none: 0) and has the value 0."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    q, k, v = randn(rows, H, D), randn(n, Hk, D), randn(n, Hk, D) * size
    if mass:
        u = torch.ones(D, device="cuda")
        u[1::2] = -1
        q = q - (q @ u)[..., None] * u / D + 0.5 * u
        k = k - (k @ u)[..., None] * u / D
        k[0] = u * (math.log(n * mass / (1 - mass)) + 0.5) / (0.5 * D ** 0.5)
        v[0] = 0
    return q, k, v


def _within(got, ref, var, dtype, roundings):
    tol = (((U[dtype] + 2.0 ** -12) * ref.abs()) ** 2 + (roundings * var) ** 2).sqrt()
    if dtype == "f16":
        tol = tol + 2.0 ** -25
    assert got.isfinite().all() and got.numel() >= 1000
    assert _rms(got.double() - ref) <= 2 * _rms(tol), (_rms(got.double() - ref), _rms(tol), _rms(ref))


# ------------------------------------------------------------ the 4-bit cache
def _cache(k, v, requests):
    """A pool that holds k, v once, and a table by which every request has them."""
    import torch
    n, Hk, D = k.shape
    pages = (n + 63) // 64
    pool = mb.kv4_pool(pages, Hk, D)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    mb.kv4_append(pool, k, v, slots)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(requests, 1)
    return (pool, table, *mb.kv4_read(pool, slots, D, torch.float32))


def _kv4(q, pool, table, n, each):
    """`each` new tokens of every request, all over n tokens."""
    import torch
    B = table.shape[0]
    cu = torch.arange(0, B * each + 1, each, dtype=torch.int32, device="cuda")
    return mb.kv4_attention(q, pool, table, torch.full((B,), n, dtype=torch.int32, device="cuda"), cu)


def _check_kv4(k, v, q, dtype, requests, each):
    import torch
    q = q.to(torch.float16 if dtype == "f16" else torch.bfloat16)
    pool, table, kc, vc = _cache(k, v, requests)
    n = k.shape[0]
    got = _kv4(q, pool, table, n, each)
    see = n - each + 1 + torch.arange(requests * each, device="cuda") % each
    ref, var = _exact(q, kc, vc, see, q.shape[2] ** -0.5)
    _within(got, ref, var, dtype, 2.0 ** -11 * (2 ** 0.5 if dtype == "bf16" else 1))
    return got


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("requests,each", [(3, 1), (700, 1), (130, 6)],
                         ids=["few", "many", "rows"])  # parts of a request; a request a warp; 16-row blocks
@pytest.mark.parametrize("size,mass", [(1.0, 0.9), (0.1, 0.9), (0.01, 0.9), (1e-3, 0.5), (1e-4, 0), (0.1, 0.99),
                                       (300.0, 0.9), (3e4, 0.5)])
def test_kv4_attention_small_weights(dtype, D, requests, each, size, mass):
    n, H, Hk = 4700, 8, 2
    q, k, v = _inputs(n, requests * each, H, Hk, D, size, mass, int(size * 1e4) + D)
    _check_kv4(k, v, q, dtype, requests, each)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sizes", [(1e-4, 0.01, 1.0, 100.0), (100.0, 1.0, 0.01, 1e-4), (1e-3, 50.0, 1e-3, 50.0)],
                         ids=["growing", "falling", "alternating"])
def test_kv4_attention_values_that_change_along_the_context(dtype, D, sizes):
    import torch
    n = 3000
    q, k, v = _inputs(n, 400, 8, 2, D, 1.0, 0, 5)
    v *= torch.tensor(sizes, device="cuda")[torch.arange(n, device="cuda") * len(sizes) // n][:, None, None]
    _check_kv4(k, v, q, dtype, 400, 1)


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_kv4_attention_what_lies_behind_a_request_changes_nothing(dtype, D):
    """Slots behind the last token may hold any values, large ones too."""
    import torch
    n = 1000
    q, k, v = _inputs(n + 20, 40, 8, 2, D, 0.01, 0.9, 6)
    q = q.to(torch.float16 if dtype == "f16" else torch.bfloat16)
    results = []
    for behind in (0.0, 1.0, 4e5, float("inf"), float("nan")):
        k[n:], v[n:] = behind, behind
        pool, table, _, _ = _cache(k, v, 40)
        results.append(_kv4(q, pool, table, n, 1))
    assert results[0].isfinite().all() and (results[0] != 0).any()
    for other in results[1:]:
        assert torch.equal(other, results[0])


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_kv4_attention_a_block_of_infinite_scale(D):
    """A visible block without a finite scale takes its own 32 dimensions along, and no others."""
    import torch
    n = 900
    q, k, v = _inputs(n, 40, 8, 2, D, 0.01, 0.9, 7)
    v[500, :, 3] = float("inf")
    q = q.bfloat16()
    pool, table, kc, vc = _cache(k, v, 40)
    got = _kv4(q, pool, table, n, 1)
    assert not got[..., :32].isfinite().any()
    ref, var = _exact(q, kc, vc.nan_to_num(0, 0, 0), torch.full((40,), n, device="cuda"), D ** -0.5)
    _within(got[..., 32:], ref[..., 32:], var[..., 32:], "bf16", 2.0 ** -11 * 2 ** 0.5)


@gpu
def test_kv4_attention_alone_and_among_others():
    """A request alone is cut into other parts than among many: both are within
    the same bound, so they differ by twice that at most."""
    import torch
    n, D = 4700, 128
    q, k, v = _inputs(n, 300, 8, 2, D, 0.02, 0.9, 8)
    q = q.bfloat16()
    pool, table, kc, vc = _cache(k, v, 300)
    many = _kv4(q, pool, table, n, 1)
    alone = torch.cat([_kv4(q[i:i + 1], pool, table[i:i + 1], n, 1) for i in range(20)])
    ref, var = _exact(q[:20], kc, vc, torch.full((20,), n, device="cuda"), D ** -0.5)
    for got in (many[:20], alone):
        _within(got, ref, var, "bf16", 2.0 ** -11 * 2 ** 0.5)


# ----------------------------------------------------------- packed prompts
@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 64), (8, 2, 128), (3, 3, 128)])
@pytest.mark.parametrize("n,size,mass", [(4700, 1.0, 0.9), (4700, 1.0, 0.99), (4700, 0.01, 0.99), (20001, 1.0, 0.9),
                                         (4700, 100.0, 0)])
def test_prompt_attention_small_weights(dtype, H, Hk, D, n, size, mass):
    """The last 300 tokens of a prompt behind a prefix."""
    import torch
    T = 300
    q, k, v = (x.to(torch.float16 if dtype == "f16" else torch.bfloat16)
               for x in _inputs(n, T, H, Hk, D, size, mass, n + D))
    cu = lambda m: torch.tensor([0, m], dtype=torch.int32, device="cuda")  # noqa: E731
    got = mb.prompt_attention(q, k, v, cu(T), cu(n))
    ref, var = _exact(q, k, v, n - T + 1 + torch.arange(T, device="cuda"), D ** -0.5)
    _within(got, ref, var, dtype, U[dtype])
