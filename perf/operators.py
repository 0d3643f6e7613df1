"""Cases for the paged serving operators: block tables and slot maps, rotary
positions, the 4-bit KV cache (append, read back, attention) and attention
over packed prompts.

``run`` computes a case in its plain form (elementary torch operations in 32
bits) or, with ``own`` set, through ``modelc_b200``.  Both take what
``prepare`` gives.  Sequence lengths belong to the case; the seed makes the
values, the page order and the free list.
"""
import math
import random

import torch

own = False

PAGE = 64  # tokens of a page of the 4-bit cache
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of eight requests: one new token each, the smallest
        # call (pure latency)
        {"name": "slots-decode", "op": "slots", "B": 8, "kv": 4000, "q": 1, "pad": 0},
        # a server's step that admits many ragged prompts beside running
        # requests, the output padded to the captured size
        {"name": "slots-mixed", "op": "slots", "B": 700, "kv": 9000, "q": 500, "pad": 1021},
        # a decode step of eight requests at the 8B head layout
        {"name": "rope-decode", "op": "rope", "T": 8, "H": 32, "Hk": 8, "D": 128, "rot": 128,
         "layout": "half", "scaling": "llama3", "positions": 131072, "dtype": "bf16", "out": "bf16"},
        # packed prompts of the 8B layout: q and k are views of one fused
        # projection's f32 output, rounded to bf16 on the way out
        {"name": "rope-prompt", "op": "rope", "T": 16384, "H": 32, "Hk": 8, "D": 128, "rot": 128,
         "layout": "half", "scaling": "llama3", "positions": 131072, "dtype": "f32", "out": "bf16"},
        # an odd token count, interleaved pairs, half of a 64-wide head, f32
        {"name": "rope-partial", "op": "rope", "T": 1237, "H": 32, "Hk": 4, "D": 64, "rot": 32,
         "layout": "interleaved", "scaling": "yarn", "positions": 32768, "dtype": "f32", "out": "f32"},
        # a verify step's new tokens of eight requests into the cache
        {"name": "append-verify", "op": "append", "T": 40, "Hk": 8, "D": 128, "pages": 512,
         "dtype": "bf16"},
        # a whole batch of prompts into the cache, the 64-wide layout
        {"name": "append-prompt", "op": "append", "T": 16001, "Hk": 4, "D": 64, "pages": 600,
         "dtype": "f16"},
        # one request decoding after a 1024-token prompt at the 8B layout:
        # the smallest attention call
        {"name": "kv4-decode", "op": "kv4", "B": 1, "kv": 1100, "q": 1, "H": 32, "Hk": 8, "D": 128,
         "dtype": "bf16"},
        # the verify forward of 8 requests, 4 drafts and the bonus position,
        # ragged contexts
        {"name": "kv4-verify", "op": "kv4", "B": 8, "kv": 12000, "q": 5, "H": 32, "Hk": 8, "D": 128,
         "dtype": "f16"},
        # 32 long requests decoding at the 70B head layout
        {"name": "kv4-long", "op": "kv4", "B": 32, "kv": 32768, "q": 1, "H": 64, "Hk": 8, "D": 128,
         "dtype": "bf16"},
        # several short ragged prompts at the TinyLlama layout, one of them
        # after a cached prefix
        {"name": "prompt-ragged", "op": "prompt", "B": 5, "T": 1501, "prefix": 300, "H": 32, "Hk": 4,
         "D": 64, "dtype": "f16"},
        # long packed prompts at the 8B layout
        {"name": "prompt-long", "op": "prompt", "B": 2, "T": 8192, "prefix": 0, "H": 32, "Hk": 8,
         "D": 128, "dtype": "bf16"},
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(32, 4, 64), (4, 4, 64), (32, 8, 128), (64, 8, 128), (8, 1, 128), (12, 4, 64), (6, 2, 128)]


def draw(rng):
    op = rng.choice(["slots", "rope", "append", "kv4", "kv4", "prompt", "prompt"])
    H, Hk, D = rng.choice(_HEADS)
    if op == "slots":
        B = _between(rng, 1, 700)
        return {"op": op, "B": B, "kv": _between(rng, 1, 9000), "q": _between(rng, 1, 500),
                "pad": rng.choice([0, 1, 77, 1021])}
    if op == "rope":
        d, o = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
        return {"op": op, "T": max(1, _between(rng, 1, 8000) * 32 * 128 // (H * D)), "H": H, "Hk": Hk,
                "D": D, "rot": rng.choice([D, D, D // 2, D // 4]),
                "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "ntk", "llama3", "yarn"]),
                "positions": rng.choice([4096, 32768, 131072]), "dtype": d, "out": o}
    if op == "append":
        T = _between(rng, 1, 16000)
        return {"op": op, "T": T, "Hk": rng.choice([1, 2, 4, 8]), "D": rng.choice([64, 128]),
                "pages": (T + PAGE - 1) // PAGE + rng.randrange(1, 300),
                "dtype": rng.choice(["f32", "f16", "bf16"])}
    if op == "kv4":
        B = _between(rng, 1, 64)
        q = rng.choice([1, 1, 1, 2, 5, 8])
        return {"op": op, "B": B, "kv": _between(rng, 1, max(64, 32 * 16384 // (B * max(1, q // 2)))),
                "q": q, "H": H, "Hk": Hk, "D": D, "dtype": rng.choice(["f16", "bf16"])}
    T = _between(rng, 2, 3900 if H > 32 else 5500)
    return {"op": op, "B": _between(rng, 1, min(T, 40)), "T": T, "prefix": rng.choice([0, 0, 111, 500]),
            "H": H, "Hk": Hk, "D": D, "dtype": rng.choice(["f16", "bf16"])}


def _split(total, n, salt, least=1):
    """`total` in n ragged parts, by the case alone."""
    r = random.Random("%s %d %d" % (salt, total, n))
    w = [r.uniform(0.2, 1.0) for _ in range(n)]
    got = [least + int((total - n * least) * x / sum(w)) for x in w]
    got[-1] += total - sum(got)
    return got


def _lengths(c):
    """(new tokens, tokens in the cache after them or keys) of each sequence."""
    B = c["B"]
    if c["op"] == "slots":
        r = random.Random("slots %d %d %d" % (B, c["kv"], c["q"]))
        q = [r.randint(0, c["q"]) if c["q"] > 1 else 1 for _ in range(B)]
        kv = [r.randint(0, c["kv"]) for _ in range(B)]
        return q, [a + b for a, b in zip(q, kv)]
    if c["op"] == "kv4":
        r = random.Random("kv4 %d %d %d" % (B, c["kv"], c["q"]))
        q = [r.randint(1, c["q"]) if b else c["q"] for b in range(B)]
        kv = [r.randint(1 + c["kv"] // 3, c["kv"]) if b else c["kv"] for b in range(B)]
        return q, [max(a, b) for a, b in zip(q, kv)]
    q = _split(c["T"], B, "prompt")
    return q, [n + (c["prefix"] if b % 2 == 1 else 0) for b, n in enumerate(q)]


def _pairs(q, k):
    """(query, key) pairs that a causal mask leaves."""
    return sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(q, k))


def work(c):
    op = c["op"]
    if op == "slots":
        q, kv = _lengths(c)
        T = sum(q) + c["pad"]
        new = sum((k + PAGE - 1) // PAGE - (k - n + PAGE - 1) // PAGE for n, k in zip(q, kv))
        return {"bytes": 4 * (4 * c["B"] + 2 * T + 2 * new), "flops": 0}
    if op == "rope":
        n = c["T"] * (c["H"] + c["Hk"])
        rows = min(c["T"], c["positions"])
        return {"bytes": n * c["D"] * (SIZES[c["dtype"]] + SIZES[c["out"]]) + 4 * c["T"] + 4 * c["rot"] * rows,
                "flops": 3 * n * c["rot"]}
    if op == "append":
        n = 2 * c["T"] * c["Hk"] * c["D"]  # K and V, in, in 4.5 bits, and read back
        return {"bytes": 2 * n * SIZES[c["dtype"]] + 2 * n * 9 // 16 + 4 * c["T"], "flops": 4 * n}
    q, k = _lengths(c)
    qo = 2 * sum(q) * c["H"] * c["D"] * SIZES[c["dtype"]]
    if op == "kv4":
        pages = sum((n + PAGE - 1) // PAGE for n in k)
        return {"bytes": qo + 2 * sum(k) * c["Hk"] * c["D"] * 9 // 16 + 4 * pages,
                "flops": 4 * c["H"] * c["D"] * _pairs(q, k)}
    return {"bytes": qo + 2 * sum(k) * c["Hk"] * c["D"] * SIZES[c["dtype"]],
            "flops": 4 * c["H"] * c["D"] * _pairs(q, k)}


# ------------------------------------------------------------------ inputs
def _frequencies(c):
    """Angle per position of each rotated pair, and the factor of cos and sin,
    in 64 bits on the CPU (the long-context rules of the public papers)."""
    n = c["rot"] // 2
    theta, factor, old = 500000.0, 8.0, 8192.0
    i = torch.arange(n, dtype=torch.float64)
    f = theta ** (-2.0 * i / c["rot"])
    if c["scaling"] == "linear":
        return f / factor, 1.0
    if c["scaling"] == "ntk":
        base = theta * factor ** (c["rot"] / max(c["rot"] - 2, 1))
        return base ** (-2.0 * i / c["rot"]), 1.0
    if c["scaling"] == "llama3":
        turns = old * f / (2 * math.pi)  # whole turns over the old context
        smooth = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * (smooth + (1 - smooth) / factor), 1.0
    if c["scaling"] == "yarn":
        where = lambda turns: c["rot"] * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(where(32.0)), 0), min(math.ceil(where(1.0)), c["rot"] - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _cu(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    perm = lambda n: torch.randperm(n, generator=g, device="cuda").to(torch.int32)  # noqa: E731
    op, s = c["op"], {"case": c}
    if op == "slots":
        q, kv = _lengths(c)
        have = [(k - n + PAGE - 1) // PAGE for n, k in zip(q, kv)]
        need = [(k + PAGE - 1) // PAGE for k in kv]
        width, n_pages = max(need) + 3, sum(need) + 50
        order = perm(n_pages)
        table = torch.full((c["B"], width), -1, dtype=torch.int32, device="cuda")
        held = torch.arange(width, device="cuda")[None] < torch.tensor(have, device="cuda")[:, None]
        table[held] = order[:sum(have)]
        free = order[sum(have):].contiguous()
        s.update(kv_len=torch.tensor([k - n for n, k in zip(q, kv)], dtype=torch.int32).cuda(),
                 q_len=torch.tensor(q, dtype=torch.int32).cuda(), table=table, free=free,
                 n_free=torch.tensor([free.numel()], dtype=torch.int32).cuda(),
                 tokens=sum(q) + c["pad"])
    elif op == "rope":
        f, factor = _frequencies(c)
        at = torch.arange(c["positions"], dtype=torch.float64, device="cuda")[:, None] * f.cuda()
        H, Hk, D = c["H"], c["Hk"], c["D"]
        qkv = randn(c["T"], (H + 2 * Hk) * D).to(DTYPES[c["dtype"]])  # one fused projection
        s.update(cos=(at.cos() * factor).float(), sin=(at.sin() * factor).float(),
                 q=qkv[:, :H * D].unflatten(1, (H, D)),
                 k=qkv[:, H * D:(H + Hk) * D].unflatten(1, (Hk, D)),
                 positions=torch.randint(0, c["positions"], (c["T"],), generator=g, device="cuda",
                                         dtype=torch.int32))
    elif op == "append":
        T, Hk, D = c["T"], c["Hk"], c["D"]
        kv = randn(2, T, Hk, D) * (0.5 + randn(1, 1, Hk, D).abs())  # channels of different size
        slots = torch.arange((T + PAGE - 1) // PAGE * PAGE, dtype=torch.int32, device="cuda")
        pages = perm(c["pages"])[: slots.numel() // PAGE]
        slots = (pages.repeat_interleave(PAGE) * PAGE + slots % PAGE)[:T].to(torch.int32)
        s.update(k=kv[0].to(DTYPES[c["dtype"]]), v=kv[1].to(DTYPES[c["dtype"]]), slots=slots,
                 pool=torch.zeros((c["pages"], Hk, 72 * D), dtype=torch.uint8, device="cuda"))
    elif op == "kv4":
        q, kv = _lengths(c)
        H, Hk, D = c["H"], c["Hk"], c["D"]
        need = [(n + PAGE - 1) // PAGE for n in kv]
        n_pages = sum(need) + 7
        order = perm(n_pages)
        table = torch.full((c["B"], max(need) + 1), -1, dtype=torch.int32, device="cuda")
        held = torch.arange(table.shape[1], device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
        table[held] = order[:sum(need)]
        pool = torch.empty((n_pages, Hk, 72 * D), dtype=torch.uint8, device="cuda")
        size = 0.5 + randn(1, Hk, D).abs()  # channels of different size
        for p in range(0, n_pages, 512):
            n = min(512, n_pages - p) * PAGE
            _store(pool, randn(n, Hk, D) * size, randn(n, Hk, D),
                   torch.arange(p * PAGE, p * PAGE + n, device="cuda"))
        s.update(q=(randn(sum(q), H, D) * 1.5).to(DTYPES[c["dtype"]]), pool=pool, table=table, cu_q=_cu(q),
                 kv_len=torch.tensor(kv, dtype=torch.int32).cuda())
    else:
        q, kv = _lengths(c)
        dt = DTYPES[c["dtype"]]
        s.update(q=(randn(sum(q), c["H"], c["D"]) * 1.5).to(dt), k=randn(sum(kv), c["Hk"], c["D"]).to(dt),
                 v=randn(sum(kv), c["Hk"], c["D"]).to(dt), cu_q=_cu(q), cu_k=_cu(kv))
    return s


# ------------------------------------------- the 4-bit page format (plain)
# A page holds 64 tokens of one key/value head in 72 D bytes: K codes (64 rows
# of D/2 bytes), V codes, K scales, V scales (f16).  A row is D/32 q4_0 blocks
# of 32 values: value = (code - 8) * scale.  Its D/8 words of 32 bits hold the
# code of value d in word d % (D/8), nibble PLACE[d // (D/8)]; rows of D = 128
# swap their two halves where bit 1 of the token is set.  Scales are ordered
# [8 groups of 8 tokens][4][D/32][2]: entry (t, b, e) is block b of token
# ORDER[2t + e] of the group.
PLACE = (0, 4, 1, 5, 2, 6, 3, 7)
ORDER = (0, 1, 2, 3, 5, 4, 7, 6)


def _quantise(x):
    """q4_0 codes [.., D] and f16 scales [.., D/32] of x [.., D]."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.gather(-1, b.abs().argmax(-1, keepdim=True))  # of largest size, the first one
    d = top / -8.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    code = (b * inv + 8.5).trunc().clamp(0, 15).to(torch.int32)
    return code.flatten(-2), d[..., 0].half()


def _store(pool, k, v, slots):
    """The rows k, v [T, Hk, D] into their slots of the pool."""
    D = k.shape[-1]
    W = D // 8
    page, at = slots.long() // PAGE, slots.long() % PAGE
    code, d = _quantise(torch.stack([k, v], 2))  # [T, Hk, 2, D]
    shift = 4 * torch.tensor(PLACE, device=k.device)
    words = (code.unflatten(-1, (8, W)).long() << shift[:, None]).sum(-2)  # [T, Hk, 2, W]
    rows = torch.stack([(words >> s) & 255 for s in (0, 8, 16, 24)], -1).to(torch.uint8).flatten(-2)
    if D == 128:
        swapped = rows.unflatten(-1, (2, 32)).flip(-2).flatten(-2)
        rows = torch.where((at & 2).bool()[:, None, None, None], swapped, rows)
    pool[:, :, : 64 * D].unflatten(-1, (2, PAGE, D // 2))[page, :, :, at] = rows
    place = torch.tensor(ORDER, device=k.device)[at % 8]
    scales = pool[:, :, 64 * D:].unflatten(-1, (2, 8, 4, D // 32, 2, 2))
    scales[page, :, :, at // 8, place // 2, :, place % 2] = d.unsqueeze(-1).view(torch.uint8)


def _load(pages, D):
    """K and V values [.., 64, D] (f32) of pages [.., 72 D]."""
    W = D // 8
    rows = pages[..., : 64 * D].unflatten(-1, (2, PAGE, D // 2))
    if D == 128:
        swapped = rows.unflatten(-1, (2, 32)).flip(-2).flatten(-2)
        odd = (torch.arange(PAGE, device=pages.device) & 2).bool()[:, None]
        rows = torch.where(odd, swapped, rows)
    byte = rows.unflatten(-1, (W, 4))
    code = torch.stack([(byte[..., p // 2] >> (4 * (p % 2))) & 15 for p in PLACE], -2).flatten(-2)
    d = pages[..., 64 * D:].contiguous().view(torch.float16).unflatten(-1, (2, 8, 4, D // 32, 2))
    d = d.transpose(-1, -2).flatten(-3, -2)[..., list(ORDER), :].flatten(-3, -2).float()
    x = (code.float() - 8).unflatten(-1, (D // 32, 32)) * d[..., None]
    x = x.flatten(-2)
    return x.select(-3, 0), x.select(-3, 1)


# -------------------------------------------------------------- plain forms
def _plain_slots(s):
    kv, q, table, free, T = s["kv_len"], s["q_len"], s["table"], s["free"], s["tokens"]
    new = kv + q
    have, need = (kv + PAGE - 1) // PAGE, (new + PAGE - 1) // PAGE
    start = (need - have).cumsum(0) - (need - have)
    j = torch.arange(table.shape[1], device=kv.device)[None]
    nth = start[:, None] + j - have[:, None]
    fresh = (j >= have[:, None]) & (j < need[:, None])
    last = (s["n_free"][0] - 1 - nth).long()
    page = torch.where(last >= 0, free[last.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where(fresh, page, table))
    cu = torch.cat([torch.zeros_like(q[:1]), q.cumsum(0).to(torch.int32)])
    t = torch.arange(T, device=kv.device, dtype=torch.int32)
    z = torch.searchsorted(cu[1:], t, right=True).clamp(max=q.numel() - 1)
    pos = kv[z] + t - cu[z]
    page = table[z, (pos // PAGE).clamp(max=table.shape[1] - 1).long()]
    live = t < cu[-1]
    slots = torch.where(live & (page >= 0), page * PAGE + pos % PAGE, -1)
    return {"cu_q": cu, "positions": torch.where(live, pos, 0).to(torch.int32),
            "slots": slots.to(torch.int32), "new_len": new,
            "n_free": (s["n_free"] - (need - have).sum()).to(torch.int32), "table": table}


def _turn(x, cos, sin, rot, layout, out):
    x = x.float()
    a, rest = x[..., :rot], x[..., rot:]
    if layout == "half":
        x0, x1 = a[..., : rot // 2], a[..., rot // 2:]
        y = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)
    else:
        x0, x1 = a[..., 0::2], a[..., 1::2]
        y = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
    return torch.cat([y, rest], -1).to(out)


def _plain_rope(s):
    c = s["case"]
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    return {n: _turn(s[n], cos, sin, c["rot"], c["layout"], DTYPES[c["out"]]) for n in ("q", "k")}


def _plain_append(s):
    D = s["case"]["D"]
    _store(s["pool"], s["k"], s["v"], s["slots"])
    page, at = s["slots"].long() // PAGE, s["slots"].long() % PAGE
    first = page.unique()  # only the pages that were written
    k, v = _load(s["pool"][first], D)  # [pages, Hk, 64, D]
    i = torch.searchsorted(first, page)
    return {"k": k[i, :, at].to(s["k"].dtype), "v": v[i, :, at].to(s["v"].dtype)}


def _softmax_rows(x, mask):
    """Softmax over the last axis where mask is true; rows without one are 0."""
    x = x.masked_fill(~mask, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = (x - top.masked_fill(top == -math.inf, 0)).exp()
    return e / e.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_kv4(s):
    c, q, table, cu = s["case"], s["q"], s["table"], s["cu_q"].long()
    B, H, Hk, D, n = c["B"], c["H"], c["Hk"], c["D"], c["q"]
    k, v = _load(s["pool"][table.clamp(min=0).long()], D)  # [B, pages, Hk, 64, D]
    k, v = (x.transpose(1, 2).flatten(2, 3) for x in (k, v))  # [B, Hk, L, D]
    j = torch.arange(n, device=q.device)
    at = (cu[:-1, None] + j).clamp(max=q.shape[0] - 1)  # [B, n] rows of q, some of the next request
    qf = q[at].float().unflatten(2, (Hk, H // Hk)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    x = (qf @ k.transpose(2, 3)) / math.sqrt(D)  # [B, Hk, G n, L]
    lens, rows = s["kv_len"].long(), cu[1:] - cu[:-1]
    where = lens[:, None] - rows[:, None] + j  # a row's own position
    mask = torch.arange(k.shape[2], device=q.device) <= where[..., None]  # [B, n, L]
    p = _softmax_rows(x.unflatten(2, (-1, n)), mask[:, None, None]).flatten(2, 3)
    o = (p @ v).unflatten(2, (-1, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, n, H, D]
    return o[j < rows[:, None]].to(q.dtype)


def _packed(cu, n, device):
    """Sequence and place in it of packed rows."""
    t = torch.arange(n, device=device)
    z = torch.searchsorted(cu[1:].long(), t, right=True)
    return z, t - cu.long()[z]


def _plain_prompt(s):
    q, k, v, cu_q, cu_k = s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"]
    G = q.shape[1] // k.shape[1]
    zq, iq = _packed(cu_q, q.shape[0], q.device)
    zk, ik = _packed(cu_k, k.shape[0], q.device)
    lens = (cu_k[1:] - cu_k[:-1] - cu_q[1:] + cu_q[:-1]).long()  # keys before the first query
    mask = (zq[:, None] == zk) & (ik <= (iq + lens[zq])[:, None])
    qf = q.float().transpose(0, 1).unflatten(0, (-1, G))  # [Hk, G, Tq, D]
    kf, vf = (x.float().transpose(0, 1)[:, None] for x in (k, v))
    p = _softmax_rows((qf @ kf.transpose(2, 3)) / math.sqrt(q.shape[2]), mask)
    return (p @ vf).flatten(0, 1).transpose(0, 1).to(q.dtype).contiguous()


def _own(s):
    import modelc_b200 as mb
    c = s["case"]
    op = c["op"]
    if op == "slots":
        step = mb.paged_slots(s["kv_len"], s["q_len"], s["table"], s["free"], s["n_free"], s["tokens"], PAGE)
        return {"cu_q": step.cu_q, "positions": step.positions, "slots": step.slots,
                "new_len": step.new_len, "n_free": step.n_free, "table": s["table"]}
    if op == "rope":
        q, k = mb.rope(s["q"], s["k"], s["positions"], s["cos"], s["sin"], layout=c["layout"],
                       dtype=DTYPES[c["out"]])
        return {"q": q, "k": k}
    if op == "append":
        mb.kv4_append(s["pool"], s["k"], s["v"], s["slots"])
        k, v = mb.kv4_read(s["pool"], s["slots"], c["D"], s["k"].dtype)
        return {"k": k, "v": v}
    if op == "kv4":
        return mb.kv4_attention(s["q"], s["pool"], s["table"], s["kv_len"], s["cu_q"])
    return mb.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"])


PLAIN = {"slots": _plain_slots, "rope": _plain_rope, "append": _plain_append, "kv4": _plain_kv4,
         "prompt": _plain_prompt}


def run(s):
    return _own(s) if own else PLAIN[s["case"]["op"]](s)


# ------------------------------------------------------------- in 64 bits
def _exact_attention(q, k, v, first):
    """Rows q [n, H, D] at positions first.. over keys k, v [L, Hk, D]."""
    n, H, D = q.shape
    out = torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    key = torch.arange(k.shape[0], device=q.device)
    for h in range(H):
        kh, vh = k[:, h * k.shape[1] // H].double(), v[:, h * k.shape[1] // H].double()
        for r in range(0, n, 4096):
            row = torch.arange(r, min(n, r + 4096), device=q.device)
            x = q[row, h].double() @ kh.T * D ** -0.5
            x = x.masked_fill(key > (row + first)[:, None], -math.inf)
            out[row, h] = torch.where((row + first >= 0)[:, None], x.softmax(-1) @ vh, 0.0)
    return out


def _exact_pages(pages, D):
    """K and V [pages * 64, Hk, D] in 64 bits, word by word."""
    n, Hk = pages.shape[:2]
    W = D // 8
    out = torch.empty(2, n, PAGE, Hk, D, dtype=torch.float64, device=pages.device)
    words = pages[:, :, : 64 * D].contiguous().view(torch.int32).view(n, Hk, 2, PAGE, W).permute(2, 0, 3, 1, 4)
    f16 = pages[:, :, 64 * D:].contiguous().view(torch.float16).view(n, Hk, 2, 8, 4, D // 32, 2)
    for tok in range(PAGE):
        x = words[:, :, tok]  # [2, n, Hk, W]
        if D == 128 and tok & 2:
            x = torch.roll(x, W // 2, -1)
        e = ORDER.index(tok % 8)
        for i in range(8):
            code = (x >> (4 * PLACE[i])) & 15
            block = (torch.arange(W, device=pages.device) + i * W) // 32
            d = f16[:, :, :, tok // 8, e // 2, :, e % 2].permute(2, 0, 1, 3)[..., block].double()
            out[:, :, tok, :, i * W:(i + 1) * W] = (code - 8).double() * d
    return out.flatten(1, 2)


def exact(c, seed):
    op = c["op"]
    if op == "slots":
        return None  # whole numbers
    s = prepare(c, seed)
    if op == "rope":
        f, factor = _frequencies(c)
        at = s["positions"].double()[:, None, None] * f.cuda()
        turn = torch.polar(torch.full_like(at, factor), at)
        got = {}
        for name in ("q", "k"):
            x = s[name].double()
            a, rest = x[..., : c["rot"]], x[..., c["rot"]:]
            pair = a.unflatten(-1, (2, -1)).transpose(-1, -2) if c["layout"] == "half" else a.unflatten(-1, (-1, 2))
            z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
            z = z.transpose(-1, -2).flatten(-2) if c["layout"] == "half" else z.flatten(-2)
            got[name] = torch.cat([z, rest], -1)
        return got
    if op == "append":
        got = {}
        for name in ("k", "v"):
            b = s[name].double().view(*s[name].shape[:2], -1, 32)
            low, high = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
            first = b.abs().argmax(-1, keepdim=True)
            top = torch.where(b.gather(-1, first) > 0, high, low)
            d = -top / 8
            code = torch.where(d == 0, 8.0, (b / d + 8.5).floor().clamp(0, 15))
            got[name] = ((code - 8) * d.float().half().double()).view(s[name].shape)
        return got
    q, kv = _lengths(c)
    out, a, b = [], 0, 0
    for z, (n, m) in enumerate(zip(q, kv)):
        if op == "kv4":
            k, v = _exact_pages(s["pool"][s["table"][z, : (m + PAGE - 1) // PAGE].long()], c["D"])
            k, v = k[:m], v[:m]
        else:
            k, v = s["k"][b:b + m], s["v"][b:b + m]
        out.append(_exact_attention(s["q"][a:a + n], k, v, m - n))
        a, b = a + n, b + m
    return torch.cat(out)
