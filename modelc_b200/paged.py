"""Paged serving on torch tensors: block tables and slot maps, rotary
positions, the 4-bit KV cache and attention over it and over packed prompts.

Each function checks its tensors, allocates its outputs with torch and makes
one asynchronous call of the C ABI (include/modelc_cuda.h) on the current
stream of the tensors' device; the arithmetic is described there.  Tensors
used on another stream than the one they were allocated on need torch's usual
care (record_stream or events).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, lib

PAGE = 64  # tokens of a page of the 4-bit cache

_ACT = {torch.float32: _lib.ACT_F32, torch.float16: _lib.ACT_F16, torch.bfloat16: _lib.ACT_BF16}
_HALF = (torch.float16, torch.bfloat16)


def _index(t: torch.Tensor, name: str, device, shape=None) -> int:
    """Pointer of a contiguous int32 tensor on `device`."""
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous int32 tensor on {device} is wanted")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, {tuple(shape)} is wanted")
    return t.data_ptr()


def _heads(t: torch.Tensor, name: str, device) -> torch.Tensor:
    """[tokens, heads, head_dim] on `device` with a contiguous last axis."""
    if t.dim() != 3 or t.device != device or t.dtype not in _ACT:
        raise ValueError(f"{name}: [tokens, heads, head_dim] of f32, f16 or bf16 on {device} is wanted")
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _rows16(t: torch.Tensor):
    """f16 or bf16 rows whose every head starts at a multiple of 16 bytes (a
    copy where they do not), with their token and head strides."""
    s = t.stride()
    if s[0] <= 0 or s[1] <= 0 or (s[0] | s[1]) % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        return t, t.shape[1] * t.shape[2], t.shape[2]
    return t, s[0], s[1]


def _gpu(t: torch.Tensor, name: str):
    if not t.is_cuda:
        raise ValueError(f"{name}: a CUDA tensor is wanted")
    return t.device


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class PagedStep(NamedTuple):
    """What paged_slots gives: int32 tensors."""
    cu_q: torch.Tensor       # [requests + 1] first new token of each request
    positions: torch.Tensor  # [tokens]
    slots: torch.Tensor      # [tokens] page * page_size + offset, -1 without a page
    new_len: torch.Tensor    # [requests] kv_len + q_len
    n_free: torch.Tensor     # [1] pages left; negative: pages missing


def paged_slots(kv_len, q_len, table, free_pages, n_free, tokens: int, page_size: int = PAGE) -> PagedStep:
    """Plans a step: request z holds kv_len[z] tokens and gets q_len[z] new
    ones; missing pages come from the top of the stack free_pages[:n_free]
    and are entered into table [requests, width] in place.  ``tokens`` is the
    output's length, at least the sum of q_len (mc_paged_slots)."""
    dev = _gpu(kv_len, "kv_len")
    n = kv_len.shape[0]
    if table.dim() != 2 or table.shape[0] != n:
        raise ValueError(f"table: [{n}, width] is wanted")
    if tokens < 0:
        raise ValueError("tokens: negative")
    args = (_index(kv_len, "kv_len", dev), _index(q_len, "q_len", dev, kv_len.shape), n,
            _index(table, "table", dev), table.shape[1], _index(free_pages, "free_pages", dev),
            free_pages.numel(), _index(n_free, "n_free", dev, (1,)), page_size, tokens)
    out = torch.empty(2 * (tokens + n + 1), dtype=torch.int32, device=dev)
    step = PagedStep(*out.split_with_sizes((n + 1, tokens, tokens, n, 1)))
    check(lib().mc_paged_slots(*args, *(t.data_ptr() for t in step), dev.index, _stream(dev)))
    return step


# --------------------------------------------------------- rotary positions
@dataclass(frozen=True)
class RopeScaling:
    """Long-context rules.  kind "linear": frequencies / factor; "ntk": base
    theta * factor^(rot / (rot - 2)); "llama3": pairs that turn less than
    low_turns times over old_context are divided by factor, those above
    high_turns kept, smooth between; "yarn": the same blend by the index of
    the pair between fast and slow turns, and cos, sin times 0.1 ln factor +
    1."""
    kind: str = "none"
    factor: float = 1.0
    old_context: int = 8192
    low_turns: float = 1.0
    high_turns: float = 4.0
    fast: float = 32.0
    slow: float = 1.0


def rope_frequencies(rot: int, theta: float = 10000.0, scaling: RopeScaling | None = None):
    """(angle per position of each of the rot/2 pairs, factor of cos and sin)
    as f64 numbers."""
    s = scaling or RopeScaling()
    if rot <= 0 or rot % 2:
        raise ValueError("rot must be even and positive")
    if s.kind not in ("none", "linear", "ntk", "llama3", "yarn"):
        raise ValueError(f"unknown scaling {s.kind!r}")
    if theta <= 0 or s.factor <= 0 or s.old_context <= 0:
        raise ValueError("theta, factor and old_context must be positive")
    if s.kind == "ntk":
        theta = theta * s.factor ** (rot / max(rot - 2, 1))
    f = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    if s.kind == "linear":
        return [x / s.factor for x in f], 1.0
    if s.kind == "llama3":
        def keep(x):
            turns = s.old_context * x / (2 * math.pi)
            return min(max((turns - s.low_turns) / (s.high_turns - s.low_turns), 0.0), 1.0)
        return [x * (keep(x) + (1 - keep(x)) / s.factor) for x in f], 1.0
    if s.kind == "yarn":
        def where(turns):
            return rot * math.log(s.old_context / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(where(s.fast)), 0), min(math.ceil(where(s.slow)), rot - 1)
        ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(rot // 2)]
        return ([x * (1 - r) + x / s.factor * r for x, r in zip(f, ramp)],
                0.1 * math.log(s.factor) + 1.0 if s.factor > 1 else 1.0)
    return f, 1.0


def rope_table(positions: int, rot: int, theta: float = 10000.0,
               scaling: RopeScaling | None = None, device=0):
    """(cos, sin), each f32 [positions, rot/2] on the device, for ``rope``."""
    dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    f, factor = rope_frequencies(rot, theta, scaling)
    freq = torch.tensor(f, dtype=torch.float64, device=dev)
    cos = torch.empty((positions, rot // 2), dtype=torch.float32, device=dev)
    sin = torch.empty_like(cos)
    check(lib().mc_rope_table(freq.data_ptr(), len(f), positions, factor, cos.data_ptr(),
                              sin.data_ptr(), cos.device.index, _stream(cos.device)))
    return cos, sin


def rope(q, k, positions, cos, sin, layout: str = "half", dtype=None):
    """Rotates the first 2 * cos.shape[1] values of every head of q [tokens,
    heads, head_dim] and k (or None) by their positions: pairs (i, i + rot/2)
    for layout "half", (2i, 2i + 1) for "interleaved".  Returns new tensors
    of ``dtype``, the inputs' own by default, or any for f32 inputs."""
    dev = _gpu(q, "q")
    q = _heads(q, "q", dev)
    T, H, D = q.shape
    if layout not in ("half", "interleaved"):
        raise ValueError(f"unknown layout {layout!r}")
    if cos.shape != sin.shape or cos.dim() != 2 or cos.dtype != torch.float32 or sin.dtype != torch.float32 \
            or not (cos.is_contiguous() and sin.is_contiguous()) or cos.device != dev or sin.device != dev:
        raise ValueError(f"cos, sin: contiguous f32 [positions, rot/2] on {dev} are wanted")
    dtype = dtype or q.dtype
    if dtype not in _ACT:
        raise ValueError("dtype: f32, f16 or bf16 is wanted")
    pos = _index(positions, "positions", dev, (T,))
    qo = torch.empty((T, H, D), dtype=dtype, device=dev)
    ko, Hk, kp, ks = None, 0, None, (0, 0, 0)
    if k is not None:
        k = _heads(k, "k", dev)
        if k.shape[0] != T or k.shape[2] != D or k.dtype != q.dtype:
            raise ValueError("k: q's tokens, head dim and type are wanted")
        Hk, ks, kp = k.shape[1], k.stride(), k.data_ptr()
        ko = torch.empty((T, Hk, D), dtype=dtype, device=dev)
    qs = q.stride()
    check(lib().mc_rope(q.data_ptr(), qs[0], qs[1], H, kp, ks[0], ks[1], Hk, _ACT[q.dtype], T, D,
                        2 * cos.shape[1], layout == "interleaved", pos, cos.data_ptr(),
                        sin.data_ptr(), cos.shape[0], qo.data_ptr(),
                        ko.data_ptr() if ko is not None else None, _ACT[dtype], dev.index,
                        _stream(dev)))
    return qo, ko


# -------------------------------------------------------------- 4-bit cache
def kv4_pool(n_pages: int, n_kv_heads: int, head_dim: int, device=0) -> torch.Tensor:
    """An empty pool of the 4-bit cache: uint8 [n_pages, n_kv_heads, bytes of
    a page of 64 tokens of one head]."""
    n = lib().mc_kv4_page_bytes(head_dim)
    if n == 0:
        raise ValueError(f"head dim {head_dim}: 64 or 128 is wanted")
    dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    return torch.zeros((n_pages, n_kv_heads, n), dtype=torch.uint8, device=dev)


def _pool(pool: torch.Tensor, head_dim: int):
    if pool.dim() != 3 or pool.dtype != torch.uint8 or not pool.is_contiguous() or not pool.is_cuda \
            or pool.shape[2] != 72 * head_dim:
        raise ValueError("pool: a contiguous uint8 [pages, kv heads, 72 * head_dim] CUDA tensor is wanted")
    return pool.device


def kv4_append(pool, k, v, slots) -> None:
    """Quantizes k, v [tokens, kv heads, head_dim] into their slots of the
    pool (q4_0 blocks of 32 values); slots outside the pool are skipped."""
    dev = _pool(pool, k.shape[-1])
    k, v = _heads(k, "k", dev), _heads(v, "v", dev)
    T, Hk, D = k.shape
    if v.shape != k.shape or v.dtype != k.dtype or Hk != pool.shape[1]:
        raise ValueError("k, v: one shape and type, and the pool's heads, are wanted")
    ks, vs = k.stride(), v.stride()
    check(lib().mc_kv4_append(pool.data_ptr(), pool.shape[0], Hk, D, k.data_ptr(), ks[0], ks[1],
                              v.data_ptr(), vs[0], vs[1], _ACT[k.dtype],
                              _index(slots, "slots", dev, (T,)), T, dev.index, _stream(dev)))


def kv4_read(pool, slots, head_dim: int, dtype=torch.bfloat16):
    """(k, v) [tokens, kv heads, head_dim]: the values that the slots hold."""
    dev = _pool(pool, head_dim)
    if dtype not in _ACT:
        raise ValueError("dtype: f32, f16 or bf16 is wanted")
    T, Hk = slots.numel(), pool.shape[1]
    out = torch.empty((2, T, Hk, head_dim), dtype=dtype, device=dev)
    k, v = out.unbind(0)
    check(lib().mc_kv4_read(pool.data_ptr(), pool.shape[0], Hk, head_dim,
                            _index(slots, "slots", dev), T, k.data_ptr(), v.data_ptr(),
                            _ACT[dtype], dev.index, _stream(dev)))
    return k, v


def kv4_attention(q, pool, table, kv_len, cu_q, scale: float | None = None):
    """Attention of the new tokens q [tokens, heads, head_dim] (f16, bf16)
    over the cache: rows cu_q[z]..cu_q[z+1] are the last of request z's
    kv_len[z] tokens, which the pool holds already through table [requests,
    width].  ``scale`` is 1/sqrt(head_dim) by default.  Rows that see no key
    are 0."""
    dev = _gpu(q, "q")
    q = _heads(q, "q", dev)
    T, H, D = q.shape
    if _pool(pool, D) != dev:
        raise ValueError("q, pool: on different devices")
    if q.dtype not in _HALF:
        raise ValueError("q: f16 or bf16 is wanted")
    B = kv_len.shape[0]
    if table.dim() != 2 or table.shape[0] != B:
        raise ValueError(f"table: [{B}, width] is wanted")
    Hk = pool.shape[1]
    out = torch.empty((T, H, D), dtype=q.dtype, device=dev)
    ws = torch.empty(lib().mc_kv4_attention_workspace(B, D, dev.index), dtype=torch.uint8, device=dev)
    qs = q.stride()
    check(lib().mc_kv4_attention(q.data_ptr(), qs[0], qs[1], _ACT[q.dtype], T, H, pool.data_ptr(),
                                 pool.shape[0], Hk, D, _index(table, "table", dev), table.shape[1],
                                 _index(kv_len, "kv_len", dev), _index(cu_q, "cu_q", dev, (B + 1,)),
                                 B, D ** -0.5 if scale is None else scale, out.data_ptr(),
                                 ws.data_ptr(), ws.numel(), dev.index, _stream(dev)))
    return out


# --------------------------------------------------------- packed prompts
def prompt_attention(q, k, v, cu_q, cu_k=None, scale: float | None = None, causal: bool = True):
    """Attention over packed prompts: q [n_q, heads, head_dim], k, v [n_k, kv
    heads, head_dim] (f16, bf16), sequence z holding queries cu_q[z]..cu_q[z+1]
    and keys cu_k[z]..cu_k[z+1] (cu_q's by default).  Causal: its queries are
    its last tokens.  Rows that see no key are 0."""
    dev = _gpu(q, "q")
    q, k, v = _heads(q, "q", dev), _heads(k, "k", dev), _heads(v, "v", dev)
    T, H, D = q.shape
    if q.dtype not in _HALF or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k, v: one type, f16 or bf16, is wanted")
    if k.shape != v.shape or k.shape[2] != D:
        raise ValueError("k, v: one shape, with q's head dim, is wanted")
    (q, qt, qh), (k, kt, kh), (v, vt, vh) = _rows16(q), _rows16(k), _rows16(v)
    cu_k = cu_q if cu_k is None else cu_k
    B = cu_q.shape[0] - 1
    if B < 0:
        raise ValueError("cu_q: [sequences + 1] is wanted")
    out = torch.empty((T, H, D), dtype=q.dtype, device=dev)
    check(lib().mc_prompt_attention(q.data_ptr(), qt, qh, k.data_ptr(), kt, kh,
                                    v.data_ptr(), vt, vh, _ACT[q.dtype], T, k.shape[0], H,
                                    k.shape[1], D, _index(cu_q, "cu_q", dev),
                                    _index(cu_k, "cu_k", dev, (B + 1,)), B,
                                    D ** -0.5 if scale is None else scale, causal, out.data_ptr(),
                                    dev.index, _stream(dev)))
    return out
