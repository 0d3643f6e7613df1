"""Prompts with NaN or infinite values: they go where the definition says, and
cost no more than the rows that they hide in."""
import pytest

import modelc_b200 as mb

gpu = pytest.mark.gpu


def _inputs(T, H, Hk, D, dtype, seed):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = torch.float16 if dtype == "f16" else torch.bfloat16
    q, k, v = (torch.randn(T, h, D, generator=g, device="cuda").to(dt) for h in (H, Hk, Hk))
    return q, k, v


def _cu(*x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (4, 2, 128), (3, 1, 64), (3, 3, 128)])
@pytest.mark.parametrize("what", ["nan", "inf"])
def test_one_column_of_a_token(dtype, H, Hk, D, what):
    """Rows that see the token lose that column of its heads, the others none:
    the first tokens of a sequence, the last, and ones inside and at the ends of
    the tiles of 128 keys."""
    import torch
    cu, T = _cu(0, 300, 700, 750), 750
    q, k, v = _inputs(T, H, Hk, D, dtype, 3)
    clean = mb.prompt_attention(q, k, v, cu)
    row = torch.arange(T, device="cuda")
    for at in (0, 1, 100, 127, 128, 255, 256, 299, 300, 437, 699, 700, 749):
        bad = v.clone()
        bad[at, 0, 3] = float(what)
        got = mb.prompt_attention(q, k, bad, cu)
        end = next(x for x in (300, 700, 750) if at < x)
        hit = ((row >= at) & (row < end))[:, None, None] & (torch.arange(H, device="cuda") < H // Hk)[:, None] & \
            (torch.arange(D, device="cuda") == 3)
        assert not got[hit].isfinite().any()
        rest = torch.where(hit, clean, got)
        assert rest.isfinite().all()
        # a row that was computed again has unrounded weights: both forms' own bound
        err = (rest.double() - clean.double()).abs()
        assert (err <= (2.0 ** -9 if dtype == "f16" else 2.0 ** -6) * (1 + clean.double().abs())).all()
        spared = (row < max(at - 143, 0)) | (row >= end)
        assert torch.equal(got[spared], clean[spared])


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_all_or_every_other_token(dtype, D):
    import torch
    q, k, v = _inputs(500, 4, 2, D, dtype, 4)
    for step in (1, 2, 3):
        bad = v.clone()
        bad[1::step] = float("nan")
        got = mb.prompt_attention(q, k, bad, _cu(0, 500))
        _ref = mb.prompt_attention(q[:1], k[:1], v[:1], _cu(0, 1))
        assert torch.equal(got[:1], _ref) and got[1:].isnan().all()


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", ["k", "v", "column"])
def test_a_bad_token_does_not_hold_the_call_up(D, what):
    """A NaN that every row sees costs nothing: it took 900 times the clean
    call's time when each such row was computed again."""
    import torch
    T = 4096
    q, k, v = _inputs(T, 32, 8, D, "bf16", 5)
    cu = _cu(0, T)

    def best(*x):
        took = []
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            mb.prompt_attention(*x, cu)
            b.record()
            b.synchronize()
            took.append(a.elapsed_time(b))
        return min(took)

    clean = best(q, k, v)
    bad_k, bad_v = k.clone(), v.clone()
    if what == "k":
        bad_k[0] = float("nan")
    else:
        bad_v[0, :, 5 if what == "column" else slice(None)] = float("nan")
    assert best(q, bad_k, bad_v) <= 10 * clean
