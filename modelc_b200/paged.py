"""Paged serving on torch tensors: block tables and slot maps, rotary
positions, the 4-bit KV cache and attention over it and over packed prompts.

Each function checks its tensors, allocates its outputs with torch and makes
one asynchronous call of the C ABI (include/modelc_cuda.h) on the current
stream of the tensors' device; the arithmetic is described there.  Tensors
used on another stream than the one they were allocated on need torch's usual
care (record_stream or events).  The operators have no backward pass: results
of inputs that want gradients raise when these are asked for, and what
kv4_append stores carries none.

Decode steps make these calls with a few tokens each, where the host's time is
the whole cost: the argument structs are packed with ``struct`` and passed as
one pointer (0.8 us where ctypes took 2.2 us for 22 arguments), and the stream
is asked for as a number (0.1 us where the Stream object took 2.2 us).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from functools import lru_cache
from struct import Struct
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, lib

PAGE = 64  # tokens of a page of the 4-bit cache

_ACT = {torch.float32: _lib.ACT_F32, torch.float16: _lib.ACT_F16, torch.bfloat16: _lib.ACT_BF16}
_INT, _F32, _F16, _BF16 = torch.int32, torch.float32, torch.float16, torch.bfloat16

# mc_slots_args, mc_rope_args, ... in the C compiler's layout
_SLOTS = Struct("@10P5i").pack
_ROPE = Struct("@7P4q9i").pack
_APPEND = Struct("@4P5q4i").pack
_READ = Struct("@4Pq4i").pack
_ATTENTION = Struct("@7P4q7if").pack
_PROMPT = Struct("@6P6q8if").pack


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the same number without the Stream object around it
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


def _index(t: torch.Tensor, name: str, dev: int, shape=None) -> int:
    """Pointer of a contiguous int32 tensor on CUDA device `dev`."""
    if t.dtype is not _INT or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous int32 tensor on cuda:{dev} is wanted")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, {tuple(shape)} is wanted")
    return t.data_ptr()


def _length(t: torch.Tensor, name: str) -> int:
    if t.dim() != 1:
        raise ValueError(f"{name}: one axis is wanted")
    return t.shape[0]


def _heads(t: torch.Tensor, name: str, dev: int) -> torch.Tensor:
    """[tokens, heads, head_dim] on device `dev` with a contiguous last axis."""
    if t.dim() != 3 or t.get_device() != dev or t.dtype not in _ACT:
        raise ValueError(f"{name}: [tokens, heads, head_dim] of f32, f16 or bf16 on cuda:{dev} is wanted")
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _rows16(t: torch.Tensor):
    """f16 or bf16 rows whose every head starts at a multiple of 16 bytes (a
    copy where they do not), with their token and head strides."""
    s0, s1, _ = t.stride()
    if s0 <= 0 or s1 <= 0 or (s0 | s1) % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        return t, t.shape[1] * t.shape[2], t.shape[2]
    return t, s0, s1


def _gpu(t: torch.Tensor, name: str) -> int:
    dev = t.get_device()
    if dev < 0:
        raise ValueError(f"{name}: a CUDA tensor is wanted")
    return dev


def _like(t: torch.Tensor, dtype=None) -> torch.Tensor:
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


class _NoBackward(torch.autograd.Function):
    """Keeps a result in the graph of inputs that want gradients, so that asking
    for them is an error and not a silent zero."""

    @staticmethod
    def forward(ctx, name, out, *inputs):
        ctx.name = name
        return out

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError(f"{ctx.name} has no backward pass")


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
    output's length, at least the sum of q_len: tokens behind it get no slot,
    but their pages are taken and entered (mc_paged_slots)."""
    dev = _gpu(kv_len, "kv_len")
    n = _length(kv_len, "kv_len")
    if table.dim() != 2 or table.shape[0] != n:
        raise ValueError(f"table: [{n}, width] is wanted")
    if tokens < 0:
        raise ValueError("tokens: negative")
    kv = _index(kv_len, "kv_len", dev)
    q = _index(q_len, "q_len", dev, kv_len.shape)
    tab = _index(table, "table", dev)
    n_pages = _length(free_pages, "free_pages")
    free = _index(free_pages, "free_pages", dev)
    left = _index(n_free, "n_free", dev, (1,))
    out = torch.empty(2 * (tokens + n + 1), dtype=_INT, device=kv_len.device)
    p = out.data_ptr()  # cu_q, positions, slots, new_len, n_free one behind the other
    pos = p + 4 * (n + 1)
    new = pos + 8 * tokens
    check(lib().mc_paged_slots(_SLOTS(kv, q, tab, free, left, p, pos, pos + 4 * tokens, new, new + 4 * n, n,
                                      table.shape[1], n_pages, page_size, tokens), dev, _stream(dev)))
    return PagedStep(*out.unsafe_split_with_sizes((n + 1, tokens, tokens, n, 1)))


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
    if not all(0 < x < math.inf for x in (theta, s.factor, s.old_context)):
        raise ValueError("theta, factor and old_context must be positive")
    if s.kind == "llama3" and not s.low_turns < s.high_turns:
        raise ValueError("low_turns must be below high_turns")
    if s.kind == "yarn" and not (theta > 1 and 0 < s.slow <= s.fast):
        raise ValueError("yarn: theta above 1 and 0 < slow <= fast are wanted")
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
    cos = torch.empty((positions, rot // 2), dtype=_F32, device=dev)
    sin = torch.empty_like(cos)
    dev = cos.get_device()
    check(lib().mc_rope_table(freq.data_ptr(), len(f), positions, factor, cos.data_ptr(),
                              sin.data_ptr(), dev, _stream(dev)))
    return cos, sin


def rope(q, k, positions, cos, sin, layout: str = "half", dtype=None):
    """Rotates the first 2 * cos.shape[1] values of every head of q [tokens,
    heads, head_dim] and k (or None) by their positions: pairs (i, i + rot/2)
    for layout "half", (2i, 2i + 1) for "interleaved".  Returns new tensors
    of ``dtype``, the inputs' own by default, or any for f32 inputs."""
    dev = _gpu(q, "q")
    q = _heads(q, "q", dev)
    T, H, D = q.shape
    if layout != "half" and layout != "interleaved":
        raise ValueError(f"unknown layout {layout!r}")
    if cos.shape != sin.shape or cos.dim() != 2 or cos.dtype is not _F32 or sin.dtype is not _F32 \
            or not (cos.is_contiguous() and sin.is_contiguous()) or cos.get_device() != dev \
            or sin.get_device() != dev:
        raise ValueError(f"cos, sin: contiguous f32 [positions, rot/2] on cuda:{dev} are wanted")
    own = q.dtype
    dtype = dtype or own
    if dtype not in _ACT:
        raise ValueError("dtype: f32, f16 or bf16 is wanted")
    pos = _index(positions, "positions", dev, (T,))
    qo = _like(q, dtype)
    ko, Hk, kp, kop, k0, k1 = None, 0, 0, 0, 0, 0
    if k is not None:
        k = _heads(k, "k", dev)
        if k.shape[0] != T or k.shape[2] != D or k.dtype is not own:
            raise ValueError("k: q's tokens, head dim and type are wanted")
        ko = _like(k, dtype)
        Hk, kp, kop = k.shape[1], k.data_ptr(), ko.data_ptr()
        k0, k1, _ = k.stride()
    q0, q1, _ = q.stride()
    rows, half = cos.shape
    check(lib().mc_rope(_ROPE(q.data_ptr(), kp, pos, cos.data_ptr(), sin.data_ptr(), qo.data_ptr(), kop, q0, q1,
                              k0, k1, H, Hk, _ACT[own], _ACT[dtype], T, D, 2 * half, layout == "interleaved",
                              rows), dev, _stream(dev)))
    if (q.requires_grad or k is not None and k.requires_grad) and torch.is_grad_enabled():
        qo = _NoBackward.apply("rope", qo, q, k)
        ko = None if ko is None else _NoBackward.apply("rope", ko, q, k)
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


def _pool(pool: torch.Tensor, head_dim: int) -> int:
    dev = pool.get_device()
    if pool.dim() != 3 or pool.dtype is not torch.uint8 or dev < 0 or not pool.is_contiguous() \
            or pool.shape[2] != 72 * head_dim:
        raise ValueError("pool: a contiguous uint8 [pages, kv heads, 72 * head_dim] CUDA tensor is wanted")
    return dev


def kv4_append(pool, k, v, slots) -> None:
    """Quantizes k, v [tokens, kv heads, head_dim] into their slots of the
    pool (q4_0 blocks of 32 values); slots outside the pool are skipped.  No
    two tokens of one call may share a slot."""
    dev = _pool(pool, k.shape[-1] if k.dim() else 0)
    k, v = _heads(k, "k", dev), _heads(v, "v", dev)
    T, Hk, D = k.shape
    if v.shape != k.shape or v.dtype is not k.dtype or Hk != pool.shape[1]:
        raise ValueError("k, v: one shape and type, and the pool's heads, are wanted")
    k0, k1, _ = k.stride()
    v0, v1, _ = v.stride()
    check(lib().mc_kv4_append(_APPEND(pool.data_ptr(), k.data_ptr(), v.data_ptr(),
                                      _index(slots, "slots", dev, (T,)), pool.shape[0], k0, k1, v0, v1, Hk, D,
                                      _ACT[k.dtype], T), dev, _stream(dev)))


def kv4_read(pool, slots, head_dim: int, dtype=torch.bfloat16):
    """(k, v) [tokens, kv heads, head_dim]: the values that the slots hold."""
    dev = _pool(pool, head_dim)
    if dtype not in _ACT:
        raise ValueError("dtype: f32, f16 or bf16 is wanted")
    T, Hk = slots.numel(), pool.shape[1]
    k = torch.empty((T, Hk, head_dim), dtype=dtype, device=pool.device)
    v = torch.empty_like(k)
    check(lib().mc_kv4_read(_READ(pool.data_ptr(), _index(slots, "slots", dev), k.data_ptr(), v.data_ptr(),
                                  pool.shape[0], Hk, head_dim, _ACT[dtype], T), dev, _stream(dev)))
    return k, v


@lru_cache(maxsize=4096)
def _workspace_bytes(requests: int, head_dim: int, dev: int) -> int:
    n = lib().mc_kv4_attention_workspace(requests, head_dim, dev)
    if n <= 0:
        raise ValueError(f"head dim {head_dim}: 64 or 128 is wanted" if head_dim not in (64, 128)
                         else _lib.last_error())
    return n


def kv4_attention(q, pool, table, kv_len, cu_q, scale: float | None = None):
    """Attention of the new tokens q [tokens, heads, head_dim] (f16, bf16)
    over the cache: rows cu_q[z]..cu_q[z+1] are the last of request z's
    kv_len[z] tokens, which the pool holds already through table [requests,
    width].  ``scale`` is 1/sqrt(head_dim) by default.  Rows that see no key
    are 0.  Weights times value scales are rounded to f16, in bf16 calls the
    weights too; scores and sums are f32."""
    dev = _gpu(q, "q")
    q = _heads(q, "q", dev)
    T, H, D = q.shape
    if _pool(pool, D) != dev:
        raise ValueError("q, pool: on different devices")
    dt = q.dtype
    if dt is not _BF16 and dt is not _F16:
        raise ValueError("q: f16 or bf16 is wanted")
    B = _length(kv_len, "kv_len")
    if table.dim() != 2 or table.shape[0] != B:
        raise ValueError(f"table: [{B}, width] is wanted")
    pages, Hk, _ = pool.shape
    out = _like(q)
    # torch's allocator gives and takes the workspace back in the stream's order
    # (a graph's capture from the graph's memory): nothing is kept between calls.
    # Elements of q's 2-byte type: new_empty takes 1.25 us, torch.empty 1.5.
    n = _workspace_bytes(B, D, dev)
    ws = q.new_empty(n // 2)
    q0, q1, _ = q.stride()
    check(lib().mc_kv4_attention(_ATTENTION(
        q.data_ptr(), pool.data_ptr(), _index(table, "table", dev), _index(kv_len, "kv_len", dev),
        _index(cu_q, "cu_q", dev, (B + 1,)), out.data_ptr(), ws.data_ptr(), q0, q1, pages, n, _ACT[dt], T, H, Hk,
        D, table.shape[1], B, D ** -0.5 if scale is None else scale), dev, _stream(dev)))
    if q.requires_grad and torch.is_grad_enabled():
        out = _NoBackward.apply("kv4_attention", out, q)
    return out


# --------------------------------------------------------- packed prompts
def prompt_attention(q, k, v, cu_q, cu_k=None, scale: float | None = None, causal: bool = True):
    """Attention over packed prompts: q [n_q, heads, head_dim], k, v [n_k, kv
    heads, head_dim] (f16, bf16), sequence z holding queries cu_q[z]..cu_q[z+1]
    and keys cu_k[z]..cu_k[z+1] (cu_q's by default).  Causal: its queries are
    its last tokens.  Rows that see no key are 0.  Weights are rounded to the
    inputs' type; scores and sums are f32."""
    dev = _gpu(q, "q")
    q, k, v = _heads(q, "q", dev), _heads(k, "k", dev), _heads(v, "v", dev)
    T, H, D = q.shape
    dt = q.dtype
    if (dt is not _BF16 and dt is not _F16) or k.dtype is not dt or v.dtype is not dt:
        raise ValueError("q, k, v: one type, f16 or bf16, is wanted")
    Tk, Hk, _ = k.shape
    if k.shape != v.shape or k.shape[2] != D:
        raise ValueError("k, v: one shape, with q's head dim, is wanted")
    (q, q0, q1), (k, k0, k1), (v, v0, v1) = _rows16(q), _rows16(k), _rows16(v)
    cu_k = cu_q if cu_k is None else cu_k
    B = _length(cu_q, "cu_q") - 1
    if B < 0:
        raise ValueError("cu_q: [sequences + 1] is wanted")
    out = _like(q)
    check(lib().mc_prompt_attention(_PROMPT(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _index(cu_q, "cu_q", dev), _index(cu_k, "cu_k", dev, (B + 1,)),
        out.data_ptr(), q0, q1, k0, k1, v0, v1, _ACT[dt], T, Tk, H, Hk, D, B, causal,
        D ** -0.5 if scale is None else scale), dev, _stream(dev)))
    if (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        out = _NoBackward.apply("prompt_attention", out, q, k, v)
    return out
