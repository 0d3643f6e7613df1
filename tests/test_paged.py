"""The paged serving operators against plain implementations in 64 bits.

Tolerances, with u the unit roundoff of a type (f32 2^-24, f16 2^-11, bf16
2^-8) and every kernel computing in f32 or better unless said:
  rotary positions: two products and a sum of f32-rounded factors, one
    rounding to the output: (|x0 c| + |x1 s|) 2^-22 + u |y|;
  append: exact (the same f32 operations as the weights' q4_0 rule);
  attention: scores, exponentials and sums in f32 (2^-12 covers them at these
    sizes), weights rounded to u_p for the second product (f16 over the 4-bit
    cache, the inputs' type over prompts), one rounding to the output:
    u |o| + (u_p + 2^-12) sum p |v|; f16 weights below 2^-14 lose absolute
    2^-25 each, times 8 codes: n 2^-22 at most.
"""
import ctypes as C
import math
import random

import numpy as np
import pytest

import modelc_b200 as mb
from modelc_b200 import _lib
from modelc_b200.model import dequant_q4_0, quantize_q4_0

gpu = pytest.mark.gpu

U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _torch():
    import torch
    return torch, {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    torch, _ = _torch()
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return lambda *s: torch.randn(s, generator=g, device="cuda")


def _cu(lens):
    torch, _ = _torch()
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _close(got, ref, tol):
    torch, _ = _torch()
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist(),
                           float((got.double() - ref).abs().nan_to_num(1e9).max()))


# ------------------------------------------------------------- slot maps
def _slots_ref(kv, q, table, free, n_free, page, tokens):
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    cu, pos, slots, new, taken = [0], [], [], [], 0
    for z, (a, b) in enumerate(zip(kv, q)):
        a, b = max(a, 0), max(b, 0)
        have, need = (min((n + page - 1) // page, width) for n in (a, a + b))
        for j in range(have, need):
            i = max(n_free, 0) - 1 - taken
            table[z][j] = free[i] if i >= 0 else -1
            taken += 1
        for p in range(a, a + b):
            pg = table[z][p // page] if p // page < width else -1
            pos.append(p)
            slots.append(pg * page + p % page if pg >= 0 else -1)
        cu.append(cu[-1] + b)
        new.append(a + b)
    pad = tokens - len(pos)
    return cu, pos + [0] * pad, slots + [-1] * pad, new, n_free - taken, table


@gpu
@pytest.mark.parametrize("B,kv,q,page,pad,spare,cut", [
    (1, 0, 1, 64, 0, 0, 0), (1, 63, 1, 64, 3, 1, 0), (8, 500, 1, 64, 0, 5, 0), (5, 40, 70, 16, 9, 2, 0),
    (3, 0, 200, 1, 1, 0, 0), (33, 100, 3, 7, 0, 4, 0), (1024, 90, 2, 64, 0, 1, 0),
    (1025, 90, 5, 64, 77, 3, 0), (2500, 20, 9, 16, 1000, 3, 0), (6, 90, 300, 64, 0, 0, 5),
    (4, 10, 100, 16, 0, 0, 1000), (2, 0, 9000, 64, 0, 3, 0)])
def test_paged_slots(B, kv, q, page, pad, spare, cut):
    """Every array against a loop; `cut` pages fewer than are needed."""
    torch, _ = _torch()
    r = random.Random(B * 31 + page)
    kvs = [r.randint(0, kv) for _ in range(B)]
    qs = [r.randint(0, q) if z else q for z in range(B)]
    if B > 3:
        qs[1], kvs[2], qs[3] = 0, 0, -4
    need = [(a + max(b, 0) + page - 1) // page for a, b in zip(kvs, qs)]
    have = [(a + page - 1) // page for a in kvs]
    width = max(need) - (1 if cut else 0) + (0 if cut else 2)
    order = list(range(sum(need) + spare))
    r.shuffle(order)
    table, at = [], 0
    for h in have:
        h = min(h, width)
        table.append(order[at:at + h] + [-7] * (width - h))
        at += h
    free = order[at:]
    n_free = max(0, len(free) - spare - cut)
    tokens = sum(max(x, 0) for x in qs) + pad
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    tab = t(table)
    for _ in range(2):  # planning again gives the same step
        step = mb.paged_slots(t(kvs), t(qs), tab, t(free), t([n_free]), tokens, page)
        cu, pos, slots, new, left, ref = _slots_ref(kvs, qs, table, free, n_free, page, tokens)
        assert step.cu_q.tolist() == cu and step.new_len.tolist() == new
        assert step.positions.tolist() == pos and step.slots.tolist() == slots
        assert step.n_free.tolist() == [left] and tab.tolist() == ref


@gpu
def test_paged_slots_no_requests():
    torch, _ = _torch()
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    n = torch.tensor([3], dtype=torch.int32, device="cuda")
    step = mb.paged_slots(e, e, e.view(0, 5), e, n, 4)
    assert step.cu_q.tolist() == [0] and step.slots.tolist() == [-1] * 4
    assert step.positions.tolist() == [0] * 4 and step.n_free.tolist() == [3]


# -------------------------------------------------------- rotary positions
SCALINGS = [dict(kind="none"), dict(kind="linear", factor=4.0), dict(kind="ntk", factor=8.0),
            dict(kind="llama3", factor=8.0), dict(kind="yarn", factor=16.0, old_context=4096)]


def test_rope_frequencies():
    f, m = mb.rope_frequencies(8, 10000.0)
    assert np.allclose(f, [1, 0.1, 0.01, 0.001], rtol=1e-14) and m == 1.0
    g, _ = mb.rope_frequencies(8, 10000.0, mb.RopeScaling("linear", 4.0))
    assert np.allclose(np.array(g) * 4, f, rtol=1e-14)
    g, _ = mb.rope_frequencies(8, 10000.0, mb.RopeScaling("ntk", 8.0))
    assert g[0] == 1 and math.isclose(g[3], f[3] / 8, rel_tol=1e-12)  # the slowest pair: / factor
    g, _ = mb.rope_frequencies(128, 500000.0, mb.RopeScaling("llama3", 8.0))
    f, _ = mb.rope_frequencies(128, 500000.0)
    turns = 8192 * np.array(f) / (2 * math.pi)
    assert (np.array(g)[turns > 4] == np.array(f)[turns > 4]).all()
    assert np.allclose(np.array(g)[turns < 1], np.array(f)[turns < 1] / 8, rtol=1e-14)
    g, m = mb.rope_frequencies(128, 10000.0, mb.RopeScaling("yarn", 16.0, 4096))
    f, _ = mb.rope_frequencies(128, 10000.0)
    assert g[0] == f[0] and math.isclose(g[-1], f[-1] / 16) and math.isclose(m, 0.1 * math.log(16) + 1)
    for bad in (lambda: mb.rope_frequencies(7), lambda: mb.rope_frequencies(8, -1.0),
                lambda: mb.rope_frequencies(8, 1e4, mb.RopeScaling("what"))):
        with pytest.raises(ValueError):
            bad()


@gpu
@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["kind"])
def test_rope_table(scaling):
    s = mb.RopeScaling(**scaling)
    cos, sin = mb.rope_table(70000, 96, 500000.0, s)
    f, m = mb.rope_frequencies(96, 500000.0, s)
    at = np.arange(70000)[:, None] * np.array(f)[None]
    assert np.abs(cos.cpu().numpy() - m * np.cos(at)).max() <= m * 2.0 ** -23
    assert np.abs(sin.cpu().numpy() - m * np.sin(at)).max() <= m * 2.0 ** -23


@gpu
@pytest.mark.parametrize("types", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"),
                                   ("f16", "f16")], ids="-".join)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,Hk,D,rot,view", [
    (1, 1, 1, 64, 64, "own"), (7, 32, 8, 128, 128, "fused"), (33, 4, 4, 64, 32, "fused"),
    (5, 3, 1, 96, 24, "own"), (3, 2, 2, 64, 6, "own"), (11, 5, 0, 80, 80, "own"),
    (9, 4, 2, 128, 64, "odd"), (700, 32, 8, 128, 128, "fused"), (1201, 12, 3, 256, 128, "fused"),
    (2, 2, 1, 2, 2, "own"), (13, 6, 2, 64, 64, "tokens")])
def test_rope(types, layout, T, H, Hk, D, rot, view):
    torch, DT = _torch()
    randn = _gen(T + D)
    ti, to = DT[types[0]], DT[types[1]]
    if view == "fused":  # views of one projection's output
        x = randn(T, (H + 2 * Hk) * D).to(ti)
        q, k = x[:, :H * D].unflatten(1, (H, D)), x[:, H * D:(H + Hk) * D].unflatten(1, (Hk, D))
    elif view == "odd":  # rows that start at no multiple of a vector
        x = randn(T, (H + Hk) * D + 1).to(ti)[:, 1:]
        q, k = x[:, :H * D].unflatten(1, (H, D)), x[:, H * D:].unflatten(1, (Hk, D))
    elif view == "tokens":  # heads before tokens
        q, k = randn(H, T, D).to(ti).transpose(0, 1), randn(Hk, T, D).to(ti).transpose(0, 1)
    else:
        q, k = randn(T, H, D).to(ti), randn(T, Hk, D).to(ti) if Hk else None
    cos, sin = mb.rope_table(5000, rot, 10000.0)
    pos = torch.randint(0, 5000, (T,), device="cuda", dtype=torch.int32)
    got = mb.rope(q, k, pos, cos, sin, layout, dtype=to)
    f, _ = mb.rope_frequencies(rot)
    at = pos.double()[:, None, None] * torch.tensor(f, device="cuda", dtype=torch.float64)
    c, s = at.cos(), at.sin()
    for x, y in zip((q, k), got):
        if x is None:
            assert y is None
            continue
        x = x.double()
        a, rest = x[..., :rot], x[..., rot:]
        x0, x1 = (a[..., :rot // 2], a[..., rot // 2:]) if layout == "half" else (a[..., ::2], a[..., 1::2])
        join = (lambda u, v: torch.cat([u, v], -1)) if layout == "half" else \
            (lambda u, v: torch.stack([u, v], -1).flatten(-2))
        ref = torch.cat([join(x0 * c - x1 * s, x1 * c + x0 * s), rest], -1)
        big = torch.cat([join((x0 * c).abs() + (x1 * s).abs(), (x1 * c).abs() + (x0 * s).abs()),
                         torch.zeros_like(rest)], -1)
        assert y.dtype == to and y.is_contiguous()
        _close(y, ref, big * 2.0 ** -22 + U[types[1]] * ref.abs() + 2.0 ** -25)


@gpu
def test_rope_position_outside_the_table():
    torch, _ = _torch()
    cos, sin = mb.rope_table(16, 32)
    q = torch.ones(4, 2, 64, device="cuda")
    pos = torch.tensor([3, 16, -1, 15], device="cuda", dtype=torch.int32)
    y, _ = mb.rope(q, None, pos, cos, sin)
    assert y[[0, 3]].isfinite().all() and (y[..., 32:] == 1).all()
    assert y[1, :, :32].isnan().all() and y[2, :, :32].isnan().all()


# -------------------------------------------------------------- 4-bit cache
@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,Hk,D,view", [(1, 1, 64, "own"), (1, 8, 128, "own"), (63, 4, 64, "fused"),
                                         (64, 3, 128, "fused"), (65, 2, 128, "odd"), (130, 1, 64, "odd"),
                                         (517, 8, 128, "own"), (40, 5, 64, "tokens")])
def test_kv4_append_and_read(dtype, T, Hk, D, view):
    """Bit for bit the q4_0 rule of the weights, in any slot order."""
    torch, DT = _torch()
    randn = _gen(T * 7 + D)
    if view == "fused":
        x = randn(T, 2 * Hk * D).to(DT[dtype])
        k, v = (y.unflatten(1, (Hk, D)) for y in x.chunk(2, 1))
    elif view == "odd":
        x = randn(T, 2 * Hk * D + 1).to(DT[dtype])[:, 1:]
        k, v = (y.unflatten(1, (Hk, D)) for y in x.chunk(2, 1))
    elif view == "tokens":
        k, v = (randn(Hk, T, D).to(DT[dtype]).transpose(0, 1) for _ in range(2))
    else:
        k, v = randn(T, Hk, D).to(DT[dtype]), (randn(T, Hk, D) * 300).to(DT[dtype])
    k[0, 0, :32] = 0  # a block of zeros
    v[0, 0, :32] = torch.tensor([1.0, -1.0] * 16)  # size ties: the first decides
    v[-1, -1, 32:64] = 1e-7  # a scale that underflows
    pages = (T + 63) // 64 + 2
    pool = torch.randint(0, 255, (pages, Hk, 72 * D), device="cuda", dtype=torch.uint8)
    slots = torch.randperm(pages * 64, device="cuda")[:T].to(torch.int32)
    before = pool.clone()
    mb.kv4_append(pool, k, v, slots)
    for name, x, got in zip("kv", (k, v), mb.kv4_read(pool, slots, D, torch.float32)):
        f = x.float().cpu().numpy().reshape(-1, D)
        ref = dequant_q4_0(quantize_q4_0(f).reshape(-1, D // 32 * 18), f.shape[0], D)
        assert np.array_equal(got.cpu().numpy().reshape(-1, D), ref), name
    # every other slot is as it was
    rest = torch.tensor(sorted(set(range(pages * 64)) - set(slots.tolist())), device="cuda",
                        dtype=torch.int32)
    for a, b in zip(mb.kv4_read(pool, rest, D, torch.float32), mb.kv4_read(before, rest, D, torch.float32)):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    half = mb.kv4_read(pool, slots, D, DT[dtype])[0]
    assert torch.equal(half, mb.kv4_read(pool, slots, D, torch.float32)[0].to(DT[dtype]))


@gpu
def test_kv4_slots_outside_the_pool_and_nonfinite_blocks():
    torch, _ = _torch()
    pool = mb.kv4_pool(2, 1, 64)
    k = torch.ones(5, 1, 64, device="cuda")
    k[3, 0, 5] = float("nan")
    k[4, 0, 40] = float("-inf")
    slots = torch.tensor([-1, 128, 7, 9, 127], device="cuda", dtype=torch.int32)
    mb.kv4_append(pool, k, k, slots)
    got, _ = mb.kv4_read(pool, slots, 64, torch.float32)
    assert (got[:2] == 0).all() and (got[2] == 1).all()
    assert not got[3, 0, :32].isfinite().any() and (got[3, 0, 32:] == 1).all()
    assert got[4, 0, 40] == float("-inf") and (got[4, 0, :32] == 1).all()
    assert not got[4, 0, 32:].isfinite().any()
    seen, _ = mb.kv4_read(pool, torch.arange(128, device="cuda", dtype=torch.int32), 64)
    assert (seen != 0).any(2).sum() == 3


def _attend(q, k, v, first, scale):
    """Rows q [n, H, D] at positions first.. over k, v [L, Hk, D]: (o, sum p |v|) in 64 bits."""
    torch, _ = _torch()
    n, H, D = q.shape
    L, Hk = k.shape[:2]
    kd, vd = (x.double().repeat_interleave(H // Hk, 1) for x in (k, v))
    x = torch.einsum("nhd,lhd->hnl", q.double(), kd) * scale
    see = torch.arange(L, device=q.device)[None] <= torch.arange(n, device=q.device)[:, None] + first
    p = x.masked_fill(~see, -math.inf).softmax(-1).masked_fill(~see, 0)
    live = see.any(1)[:, None, None]
    o = torch.einsum("hnl,lhd->nhd", p.nan_to_num(), vd.nan_to_num())
    b = torch.einsum("hnl,lhd->nhd", p.nan_to_num(), vd.nan_to_num().abs())
    return torch.where(live, o, 0), torch.where(live, b, 0)


def _kv4_case(lens, Hk, D, seed, spare=3, garbage=True):
    """A pool with random tokens of each request (`lens`), all else NaN scales and codes."""
    torch, _ = _torch()
    randn = _gen(seed)
    need = [(n + 63) // 64 for n in lens]
    pages = sum(need) + spare
    pool = torch.full((max(pages, 1), Hk, 72 * D), 0xff if garbage else 0, dtype=torch.uint8, device="cuda")
    order = torch.randperm(pages, device="cpu").tolist()
    table = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32)
    at, kept = 0, []
    for z, n in enumerate(lens):
        table[z, :need[z]] = torch.tensor(order[at:at + need[z]], dtype=torch.int32)
        at += need[z]
    table = table.cuda()
    for z, n in enumerate(lens):
        k, v = randn(n, Hk, D) * (0.3 + randn(1, Hk, D).abs()), randn(n, Hk, D)
        j = torch.arange(n, device="cuda")
        slots = (table[z, j // 64] * 64 + j % 64).to(torch.int32)
        if n:
            mb.kv4_append(pool, k, v, slots)
        kept.append(mb.kv4_read(pool, slots, D, torch.float32))
    return pool, table, kept


def _check_kv4(lens, news, H, Hk, D, dtype, seed, scale=None, pad=0, amp=1.5, stride=False):
    torch, DT = _torch()
    pool, table, kept = _kv4_case(lens, Hk, D, seed)
    randn = _gen(seed + 1)
    T = sum(news) + pad
    q = (randn(T, H, D) * amp).to(DT[dtype])
    if stride:  # a view of a wider buffer, heads apart
        wide = torch.zeros(T, H, D + 8, dtype=DT[dtype], device="cuda")
        wide[..., :D] = q
        q = wide[..., :D]
    t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = mb.kv4_attention(q, pool, table, t, _cu(news), scale)
    a = 0
    for z, (n, m) in enumerate(zip(lens, news)):
        k, v = kept[z]
        ref, big = _attend(q[a:a + m], k, v, n - m, scale or D ** -0.5)
        _close(got[a:a + m], ref, U[dtype] * ref.abs() + (2.0 ** -11 + 2.0 ** -12) * big + n * 2.0 ** -22)
        a += m
    assert (got[a:] == 0).all()
    return got


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hk,D", [(4, 4, 64), (32, 4, 64), (32, 8, 128), (8, 1, 128), (6, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("lens,news", [([1], [1]), ([64], [1]), ([65], [1]), ([200], [5]), ([15, 16, 17], [1, 1, 1]),
                                       ([1000, 3, 129], [1, 3, 2]), ([700, 64, 63, 2100], [8, 1, 5, 2])],
                         ids=lambda x: "+".join(map(str, x)))
def test_kv4_attention(dtype, H, Hk, D, lens, news):
    _check_kv4(lens, news, H, Hk, D, dtype, sum(lens) + H)


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_kv4_attention_rows_without_keys(D):
    """No new tokens, no tokens at all, fewer tokens than rows, rows of no request."""
    _check_kv4([5, 0, 2, 64, 0], [0, 0, 4, 1, 2], 8, 2, D, "bf16", 5, pad=3)


@gpu
def test_kv4_attention_many_requests():
    """More requests than fit one pass over their lengths, most of them short."""
    r = random.Random(3)
    lens = [r.choice([1, 2, 63, 64, 65, 130]) for _ in range(700)]
    _check_kv4(lens, [1] * 700, 4, 2, 64, "f16", 6)


@gpu
def test_kv4_attention_long_and_many_rows():
    _check_kv4([9001], [1], 16, 2, 128, "bf16", 7)
    _check_kv4([300, 70], [70, 33], 8, 2, 128, "f16", 8)  # a chunk of a prompt


@gpu
def test_kv4_attention_scale_strides_and_peaks():
    _check_kv4([333, 20], [2, 1], 8, 2, 128, "bf16", 9, scale=0.7, amp=4.0, stride=True)
    _check_kv4([333, 20], [2, 1], 8, 2, 64, "f16", 10, scale=-0.2, stride=True)
    _check_kv4([500], [1], 4, 4, 64, "bf16", 11, scale=1e-20)


@gpu
def test_kv4_attention_deterministic_and_alone():
    """The same bits again, and for a request alone."""
    torch, _ = _torch()
    lens, news = [900, 4000, 65], [5, 5, 5]
    a = _check_kv4(lens, news, 32, 8, 128, "bf16", 12)
    assert torch.equal(a, _check_kv4(lens, news, 32, 8, 128, "bf16", 12))


@gpu
def test_kv4_attention_bad_pages_count_as_absent():
    torch, _ = _torch()
    pool, table, kept = _kv4_case([200], 2, 64, 13)
    table[0, 1] = 10 ** 6
    q = _gen(14)(1, 4, 64).half()
    got = mb.kv4_attention(q, pool, table, torch.tensor([200], dtype=torch.int32, device="cuda"), _cu([1]))
    k, v = (torch.cat([x[:64], x[128:]]) for x in kept[0])
    ref, big = _attend(q, k, v, 135, 0.125)
    _close(got, ref, U["f16"] * ref.abs() + 2.0 ** -10 * big + 200 * 2.0 ** -22)


@gpu
def test_kv4_attention_nonfinite_tokens():
    """A token's NaN reaches the rows that see it and no other."""
    torch, _ = _torch()
    for which in (0, 1):
        pool, table, _ = _kv4_case([70], 1, 64, 15)
        bad = torch.full((1, 1, 64), float("nan"), device="cuda")
        ok = torch.ones(1, 1, 64, device="cuda")
        mb.kv4_append(pool, *((bad, ok) if which == 0 else (ok, bad)), table[0, 1:2] * 64 + 4)
        q = _gen(16)(4, 2, 64).half()
        t = torch.tensor([70], dtype=torch.int32, device="cuda")
        got = mb.kv4_attention(q, pool, table, t, _cu([4]))  # rows at 66, 67, 68, 69; the token is 68
        assert got[:2].isfinite().all() and got[2:].isnan().all()


# ----------------------------------------------------------- packed prompts
def _check_prompt(lens, more, H, Hk, D, dtype, seed, causal=True, scale=None, pad=0, view="own", amp=1.5):
    torch, DT = _torch()
    randn = _gen(seed)
    keys = [max(0, n + m) for n, m in zip(lens, more)]
    Tq, Tk = sum(lens) + pad, sum(keys) + pad
    if view == "fused":
        x = (randn(Tq, (H + 2 * Hk) * D) * 1.2).to(DT[dtype])
        q, k, v = x[:, :H * D].unflatten(1, (H, D)), x[:, H * D:(H + Hk) * D].unflatten(1, (Hk, D)), \
            x[:, (H + Hk) * D:].unflatten(1, (Hk, D))
    elif view == "odd":
        q, k, v = (randn(n, h * D + 1).to(DT[dtype])[:, 1:].unflatten(1, (h, D))
                   for n, h in ((Tq, H), (Tk, Hk), (Tk, Hk)))
    elif view == "heads":
        q, k, v = (randn(h, n, D).to(DT[dtype]).transpose(0, 1) for n, h in ((Tq, H), (Tk, Hk), (Tk, Hk)))
    else:
        q, k, v = (randn(Tq, H, D) * amp).to(DT[dtype]), randn(Tk, Hk, D).to(DT[dtype]), randn(Tk, Hk, D).to(DT[dtype])
    if pad:  # what lies behind the last sequence is never read into a result
        q[sum(lens):], k[sum(keys):], v[sum(keys):] = (float("nan"),) * 3
    got = mb.prompt_attention(q, k, v, _cu(lens), _cu(keys) if any(more) else None, scale, causal)
    a = b = 0
    for n, m in zip(lens, keys):
        ref, big = _attend(q[a:a + n], k[b:b + m], v[b:b + m], m - n if causal else m, scale or D ** -0.5)
        _close(got[a:a + n], ref, U[dtype] * ref.abs() + (U[dtype] + 2.0 ** -12) * big + 2.0 ** -20)
        a, b = a + n, b + m
    assert (got[a:] == 0).all()


LENS = [[1], [2], [63], [64], [65], [127], [128], [129], [255], [256], [257], [700], [1, 1, 1], [130, 5, 0, 257, 64],
        [33] * 9]


@gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hk,D", [(4, 4, 64), (8, 1, 128), (6, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "+".join(map(str, x)))
def test_prompt_attention(dtype, H, Hk, D, lens):
    _check_prompt(lens, [0] * len(lens), H, Hk, D, dtype, sum(lens) + D)


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,more", [([5], [300]), ([1], [128]), ([200, 7], [0, 129]), ([130, 4], [-100, 60]),
                                       ([3, 300], [-3, -299]), ([257, 1, 128], [1, 1000, -1])],
                         ids=lambda x: "+".join(map(str, x)))
def test_prompt_attention_keys_and_queries_differ(D, lens, more):
    """Cached prefixes, and rows that see no key."""
    _check_prompt(lens, more, 4, 2, D, "bf16", 21)
    _check_prompt(lens, more, 4, 2, D, "f16", 22, causal=False)


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("view", ["fused", "odd", "heads"])
def test_prompt_attention_strides(D, view):
    _check_prompt([150, 40], [0, 0], 4, 2, D, "bf16", 23, view=view)


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_attention_padding_scale_and_peaks(D):
    _check_prompt([150, 40], [0, 0], 4, 2, D, "f16", 24, pad=70)
    _check_prompt([300], [0], 2, 2, D, "f16", 25, scale=2.0, amp=3.0)
    _check_prompt([300], [0], 2, 2, D, "bf16", 26, scale=-0.4, causal=False)
    _check_prompt([300], [0], 2, 2, D, "f16", 27, scale=1e-20)


@gpu
def test_prompt_attention_long():
    _check_prompt([2500, 1100], [0, 0], 4, 1, 128, "bf16", 28)
    _check_prompt([3001], [777], 2, 1, 64, "f16", 29)


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", ["nan", "inf"])
def test_prompt_attention_nonfinite_tokens(D, what):
    """A token's NaN or infinity reaches no row that does not see it, of its own sequence or another."""
    torch, _ = _torch()
    randn = _gen(30)
    lens, at = [200, 60], 100
    q, k, v = randn(260, 2, D).half(), randn(260, 1, D).half(), randn(260, 1, D).half()
    clean = mb.prompt_attention(q, k, v, _cu(lens))
    for x in (k, v):
        bad = x.clone()
        bad[at] = float(what)
        got = mb.prompt_attention(q, *((bad, v) if x is k else (k, bad)), _cu(lens))
        assert got[:at].isfinite().all() and got[200:].isfinite().all()
        _close(got[:at], clean[:at].double(), 2.0 ** -9 * (1 + clean[:at].double().abs()))
        assert torch.equal(got[200:], clean[200:])
        if x is v:
            assert not got[at:200].isfinite().any()


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_rows_before_the_first_and_behind_the_last_sequence(D):
    """Rows of no sequence are 0 wherever they lie."""
    torch, _ = _torch()
    randn = _gen(31)
    q, k, v = randn(300, 4, D).half(), randn(300, 2, D).half(), randn(300, 2, D).half()
    cu = torch.tensor([7, 200, 290], dtype=torch.int32, device="cuda")
    got = mb.prompt_attention(q, k, v, cu)
    assert (got[:7] == 0).all() and (got[290:] == 0).all()
    for a, b in ((7, 200), (200, 290)):
        ref, big = _attend(q[a:b], k[a:b], v[a:b], 0, D ** -0.5)
        _close(got[a:b], ref, U["f16"] * ref.abs() + (U["f16"] + 2.0 ** -12) * big + 2.0 ** -20)
    pool, table, kept = _kv4_case([90], 2, D, 32)
    t = torch.tensor([90], dtype=torch.int32, device="cuda")
    cu = torch.tensor([3, 5], dtype=torch.int32, device="cuda")
    got = mb.kv4_attention(q[:8], pool, table, t, cu)
    assert (got[:3] == 0).all() and (got[5:] == 0).all()
    ref, big = _attend(q[3:5], *kept[0], 88, D ** -0.5)
    _close(got[3:5], ref, U["f16"] * ref.abs() + (2.0 ** -11 + 2.0 ** -12) * big + 90 * 2.0 ** -22)


@gpu
def test_paged_slots_past_31_bits():
    """A page whose slots no int32 can name gives -1."""
    torch, _ = _torch()
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    step = mb.paged_slots(t(0, 0), t(2, 2), t(-1, -1).view(2, 1), t(5, 2 ** 30), t(2), 4, 64)
    assert step.slots.tolist() == [-1, -1, 320, 321]


# ------------------------------------------------------------------ refusals
P = 4096  # an address that no refused call reads


def _call(name, struct, device=0, **d):
    """The C entry with a struct of these fields (pointers default to P, numbers to 0)."""
    s = struct()
    for field, kind in struct._fields_:
        setattr(s, field, d.pop(field, P if kind is C.c_void_p else 0))
    assert not d, d
    return getattr(mb.lib(), name)(bytes(s), device, None)


def _struct(pointers, longs, ints, floats=""):
    class S(C.Structure):
        _fields_ = ([(n, C.c_void_p) for n in pointers.split()] + [(n, C.c_int64) for n in longs.split()] +
                    [(n, C.c_int32) for n in ints.split()] + [(n, C.c_float) for n in floats.split()])
    return S


SLOTS = _struct("kv_len q_len table free_pages n_free cu_q positions slots new_len n_free_out", "",
                "n_requests table_width n_free_pages page_size n_tokens")
ROPE = _struct("q k positions cos_table sin_table q_out k_out", "q_tok q_head k_tok k_head",
               "n_heads n_kv_heads dtype out_dtype n_tokens head_dim rot interleaved table_rows")
APPEND = _struct("pool k v slots", "n_pages k_tok k_head v_tok v_head", "n_kv_heads head_dim dtype n_tokens")
READ = _struct("pool slots k_out v_out", "n_pages", "n_kv_heads head_dim dtype n_tokens")
ATTENTION = _struct("q pool table kv_len cu_q out workspace", "q_tok q_head n_pages workspace_bytes",
                    "dtype n_tokens n_heads n_kv_heads head_dim table_width n_requests", "scale")
PROMPT = _struct("q k v cu_q cu_k out", "q_tok q_head k_tok k_head v_tok v_head",
                 "dtype n_q n_k n_heads n_kv_heads head_dim n_sequences causal", "scale")


def test_structs_match_the_header():
    """Field names and order of the packed structs are the header's."""
    import os
    import re
    from modelc_b200 import paged
    txt = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include",
                            "modelc_cuda.h")).read()
    for name, struct, pack in (("mc_slots_args", SLOTS, paged._SLOTS), ("mc_rope_args", ROPE, paged._ROPE),
                               ("mc_kv4_append_args", APPEND, paged._APPEND), ("mc_kv4_read_args", READ, paged._READ),
                               ("mc_kv4_attention_args", ATTENTION, paged._ATTENTION),
                               ("mc_prompt_args", PROMPT, paged._PROMPT)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), txt, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        kinds = {"int64_t": C.c_int64, "int32_t": C.c_int32, "float": C.c_float}
        fields = []
        for line in body.split(";")[:-1]:
            base, names = re.match(r"\s*(?:const )?(\w+)\s*(.*)", line, re.S).groups()
            for v in names.split(","):
                fields.append((v.strip().lstrip("*").strip(), C.c_void_p if "*" in v else kinds[base]))
        assert [f[0] for f in fields] == [f[0] for f in struct._fields_], name
        assert [f[1] for f in fields] == [f[1] for f in struct._fields_], name
        values = [i if k is not C.c_float else float(i) for i, (_, k) in enumerate(struct._fields_)]
        s = struct.from_buffer_copy(pack(*values) + bytes(8))
        assert [getattr(s, n) or 0 for n, _ in struct._fields_] == values, name


@pytest.mark.parametrize("status,args", [
    (-1, dict(n_requests=-1)), (-1, dict(n_tokens=-1)), (-2, dict(page_size=0)), (-1, dict(n_free=None)),
    (-1, dict(cu_q=None)), (-1, dict(kv_len=None)), (-1, dict(table=None)), (-1, dict(slots=None))])
def test_paged_slots_refuses(status, args):
    d = dict(n_requests=2, n_tokens=4, page_size=64, table_width=4, n_free_pages=4) | args
    assert _call("mc_paged_slots", SLOTS, **d) == status


@pytest.mark.parametrize("status,args", [
    (-2, dict(rot=7)), (-2, dict(rot=130)), (-2, dict(rot=0)), (-2, dict(head_dim=127)), (-3, dict(dtype=5)),
    (-3, dict(dtype=1, out_dtype=2)), (-1, dict(n_tokens=-1)), (-1, dict(q=None)), (-1, dict(k_out=None)),
    (-2, dict(table_rows=0)), (-10, dict(n_tokens=1 << 30))])
def test_rope_refuses(status, args):
    d = dict(rot=128, n_tokens=4, n_heads=8, n_kv_heads=8, head_dim=128, table_rows=10, q_tok=1024, q_head=128,
             k_tok=1024, k_head=128) | args
    assert _call("mc_rope", ROPE, **d) == status


@pytest.mark.parametrize("status,args", [
    (-2, dict(head_dim=96)), (-2, dict(n_kv_heads=0)), (-10, dict(n_pages=1 << 26)), (-1, dict(pool=4104)),
    (-3, dict(dtype=9)), (-1, dict(n_tokens=-2)), (-1, dict(slots=None))])
def test_kv4_append_and_read_refuse(status, args):
    d = dict(head_dim=128, n_kv_heads=2, n_pages=9, dtype=2, n_tokens=3) | args
    assert _call("mc_kv4_append", APPEND, **d) == status
    assert _call("mc_kv4_read", READ, **d) == status
    assert _lib.last_error()


@pytest.mark.parametrize("status,args", [
    (-2, dict(head_dim=80)), (-2, dict(n_heads=5)), (-3, dict(dtype=0)), (-1, dict(n_tokens=-1)), (-1, dict(q=None)),
    (-1, dict(scale=math.inf)), (-10, dict(n_pages=1 << 26)), (-1, dict(pool=4104)), (-1, dict(workspace=None)),
    (-1, dict(workspace=4100)), (-10, dict(n_tokens=1 << 30, n_heads=4))])
def test_kv4_attention_refuses(status, args):
    d = dict(head_dim=128, n_heads=4, n_kv_heads=2, dtype=2, n_tokens=3, scale=0.1, n_pages=9, n_requests=1,
             table_width=4, q_tok=512, q_head=128) | args
    assert _call("mc_kv4_attention", ATTENTION, **d) == status


@pytest.mark.parametrize("status,args", [
    (-2, dict(head_dim=96)), (-2, dict(n_heads=3)), (-3, dict(dtype=0)), (-1, dict(n_q=-1)), (-1, dict(v=None)),
    (-1, dict(scale=math.nan)), (-1, dict(k=4104)), (-1, dict(q_tok=260)), (-1, dict(v_head=-64)),
    (-10, dict(n_q=2 ** 31 - 1, n_heads=1024))])
def test_prompt_attention_refuses(status, args):
    d = dict(head_dim=64, n_heads=4, n_kv_heads=2, dtype=1, n_q=3, n_k=3, scale=0.1, causal=1, n_sequences=1,
             q_tok=256, q_head=64, k_tok=128, k_head=64, v_tok=128, v_head=64) | args
    assert _call("mc_prompt_attention", PROMPT, **d) == status


def test_null_struct_is_refused():
    for name in ("mc_paged_slots", "mc_rope", "mc_kv4_append", "mc_kv4_read", "mc_kv4_attention",
                 "mc_prompt_attention"):
        assert getattr(mb.lib(), name)(None, 0, None) == -1


def test_page_bytes():
    assert [mb.lib().mc_kv4_page_bytes(d) for d in (64, 128, 96, 0, -1)] == [4608, 9216, 0, 0, 0]


@gpu
def test_wrappers_refuse():
    torch, _ = _torch()
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    x = torch.zeros(4, 2, 64, device="cuda", dtype=torch.float16)
    pool = mb.kv4_pool(3, 2, 64)
    cos, sin = mb.rope_table(8, 64)
    for bad in (lambda: mb.paged_slots(i(2), i(3), i(2, 4), i(1), i(1), 4),
                lambda: mb.paged_slots(i(2), i(2), i(3, 4), i(1), i(1), 4),
                lambda: mb.paged_slots(i(2).long(), i(2), i(2, 4), i(1), i(1), 4),
                lambda: mb.rope(x, x[:3], i(4), cos, sin), lambda: mb.rope(x, x, i(3), cos, sin),
                lambda: mb.rope(x, x, i(4), cos, sin, "other"), lambda: mb.rope(x, x, i(4), cos.half(), sin),
                lambda: mb.rope(x.cpu(), x, i(4), cos, sin), lambda: mb.kv4_pool(3, 2, 96),
                lambda: mb.kv4_append(pool, x[:, :1], x[:, :1], i(4)),
                lambda: mb.kv4_append(pool, x, x.float(), i(4)),
                lambda: mb.kv4_append(pool, x.double(), x.double(), i(4)),
                lambda: mb.kv4_read(pool, i(4), 128),
                lambda: mb.kv4_attention(x.float(), pool, i(1, 3), i(1), i(2)),
                lambda: mb.kv4_attention(x, pool, i(1, 3), i(1), i(3)),
                lambda: mb.kv4_attention(x, pool, i(2, 3), i(1), i(2)),
                lambda: mb.prompt_attention(x, x, x.bfloat16(), i(2)),
                lambda: mb.prompt_attention(x, x, x[..., :32], i(2))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(mb.McError) as e:
        mb.rope(x, x, i(4), cos, sin, dtype=torch.float32)
    assert e.value.status == -3


@gpu
def test_empty_calls():
    torch, _ = _torch()
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    x = torch.zeros(0, 2, 64, device="cuda", dtype=torch.float16)
    pool = mb.kv4_pool(0, 2, 64)
    cos, sin = mb.rope_table(8, 64)
    assert mb.rope(x, x, i(0), cos, sin)[0].shape == (0, 2, 64)
    mb.kv4_append(pool, x, x, i(0))
    assert mb.kv4_read(pool, i(0), 64)[1].shape == (0, 2, 64)
    assert mb.kv4_attention(x, pool, i(0, 0), i(0), i(1)).shape == (0, 2, 64)
    assert mb.prompt_attention(x, x, x, i(1)).shape == (0, 2, 64)
    y = torch.ones(3, 2, 64, device="cuda", dtype=torch.float16)
    assert (mb.kv4_attention(y, pool, i(0, 0), i(0), i(1)) == 0).all()  # rows of no request
    assert (mb.prompt_attention(y, x, x, i(1)) == 0).all()
