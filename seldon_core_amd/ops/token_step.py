"""Operators of one step of a served token model.

A decoder's attention block between its projections, as a GPU component or a
captured module (:class:`~seldon_core_amd.models.graphed.GraphedModule`) calls
it::

    qkv = ops.lora_add(F.linear(x, w_qkv), x, A, B, tenant)     # adapters of many tenants
    q, k, v = qkv.view(T, -1, D).split((Hq, Hk, Hk), 1)
    q, k = ops.qk_norm_rope(q, k, q_norm, k_norm, positions, inv_freq)
    ops.kv_cache_write(cache, k, v, slots)                        # 16 or 8 bits
    y = ops.paged_attention(q, cache, page_table, lengths)        # one new token per request

Every op launches hand-written HIP kernels on the current stream of its
tensors' device, allocates only its outputs and workspace (from torch's
allocator, so a captured graph keeps its own) and never synchronises: lengths,
page tables, slots and adapter ids are read on the GPU only.  What the host can
see (shapes, types, strides, devices) is checked and refused with
``ValueError`` / ``TypeError``; indices that point outside a cache or a table
are left out by the kernels as each op says.  The ops are forward only.

Kernel sources: csrc/kernels/{rope,kv_cache,paged_attention,lora}.hip.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

from .._native import native

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None

if torch is not None:
    _TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3, torch.int8: 4}
    _FLOATS = (torch.float32, torch.float16, torch.bfloat16)
    _INDEX = {torch.int32: 0, torch.int64: 1}

_kernels = None


def _k():
    global _kernels
    if _kernels is None:
        _kernels = native().kernels
    return _kernels


def _tensor(t, name, dim=None, dtypes=None, device=None, contiguous=False):
    """Refuse what the kernels do not take; ``contiguous``: every stride, else only the last."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not {device}")
    if dim is not None and t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, got {tuple(t.shape)}")
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError(f"{name} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    if contiguous:
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    elif t.dim() and t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient; this operator is forward only (use torch.no_grad())")
    return t


def _launch(t, fn, *args):
    """fn(*args, stream) on the current stream of t's device."""
    d = t.device
    stream = torch.cuda.current_stream(d).cuda_stream
    if torch.cuda.current_device() == d.index:
        fn(*args, stream)
    else:
        with torch.cuda.device(d):
            fn(*args, stream)


# ------------------------------------------------------- norm and rotation
def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, *, eps: float = 1e-6, interleaved: bool = False,
                 out: Optional[Tuple] = None):
    """RMS norm of every query and key head and the rotation by its token's
    position, in one pass over both.

    ``q`` [T, Hq, D] and ``k`` [T, Hk, D] (fp32, fp16 or bf16; D even, at most
    512; any strides but a contiguous last dimension, such as views of one fused
    projection).  ``q_weight`` / ``k_weight`` [D] in q's type or fp32, or None
    for a norm without a learned weight.  ``positions`` [T] int32 or int64;
    ``inv_freq`` [R / 2] fp32 or fp64 holds the angle of each pair for one
    position, and the first R <= D dimensions turn: as pairs (i, i + R / 2), or
    (2i, 2i + 1) if ``interleaved``.  The angle is reduced in fp64, everything
    else is computed in fp32 and rounded once.

    Returns the new (q, k), contiguous, or ``out`` = (q, k), which may be the
    inputs themselves (other overlaps are not allowed).
    """
    _tensor(q, "q", 3, _FLOATS)
    dev, dt = q.device, q.dtype
    _tensor(k, "k", 3, (dt,), dev)
    T, Hq, D = q.shape
    Hk = k.shape[1]
    if k.shape[0] != T or k.shape[2] != D:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must agree in tokens and dim")
    if D < 2 or D % 2 or D > 512:
        raise ValueError(f"dim must be even, 2 to 512, got {D}")
    wf32 = None
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is None:
            continue
        _tensor(w, name, 1, (dt, torch.float32), dev, contiguous=True)
        if w.shape[0] != D:
            raise ValueError(f"{name} must have {D} values, got {w.shape[0]}")
        if wf32 is not None and wf32 != (w.dtype == torch.float32):
            raise TypeError("q_weight and k_weight must have one type")
        wf32 = w.dtype == torch.float32
    _tensor(positions, "positions", 1, _INDEX, dev, contiguous=True)
    if positions.shape[0] != T:
        raise ValueError(f"positions must have {T} values, got {positions.shape[0]}")
    _tensor(inv_freq, "inv_freq", 1, (torch.float32, torch.float64), dev, contiguous=True)
    if 2 * inv_freq.shape[0] > D:
        raise ValueError(f"inv_freq turns {2 * inv_freq.shape[0]} dimensions of {D}")
    if out is None:
        oq, ok = (torch.empty(x.shape, dtype=dt, device=dev) for x in (q, k))
    else:
        oq, ok = out
        for o, x, name in ((oq, q, "out[0]"), (ok, k, "out[1]")):
            _tensor(o, name, 3, (dt,), dev)
            if o.shape != x.shape:
                raise ValueError(f"{name} must be {tuple(x.shape)}, got {tuple(o.shape)}")
    if T and Hq + Hk:
        _launch(q, _k().qk_norm_rope, q.data_ptr(), k.data_ptr(), oq.data_ptr(), ok.data_ptr(),
                0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(), bool(wf32),
                q.stride()[:2] + k.stride()[:2] + oq.stride()[:2] + ok.stride()[:2], T, Hq, Hk, D, _TYPE[dt],
                positions.data_ptr(), _INDEX[positions.dtype], inv_freq.data_ptr(), inv_freq.dtype == torch.float64,
                inv_freq.shape[0], interleaved, eps)
    return oq, ok


# ------------------------------------------------------- paged key-value cache
class KVCache(NamedTuple):
    """The four tensors of a paged cache: ``k`` and ``v`` [pages, page size,
    heads, dim] and, where they are kept in 8 bits, their fp32 scales [pages,
    page size, heads].  Any strides but a contiguous last dimension, so the
    pages of a head may lie together too (a transposed view)."""

    k: "torch.Tensor"
    v: "torch.Tensor"
    k_scales: Optional["torch.Tensor"] = None
    v_scales: Optional["torch.Tensor"] = None


def kv_cache(pages: int, page_size: int, heads: int, dim: int, dtype=None, device="cuda") -> KVCache:
    """A zeroed cache.  ``dtype``: bf16 (the default), fp16 or fp32, or
    float8_e4m3fn or int8 for one that is quantised as it is written."""
    dtype = dtype or torch.bfloat16
    if dtype not in _TYPE:
        raise TypeError(f"dtype must be one of {[str(d) for d in _TYPE]}, got {dtype}")
    if min(pages, page_size, heads, dim) < 1:
        raise ValueError("pages, page_size, heads and dim must be positive")
    shape = (pages, page_size, heads, dim)
    k, v = torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)
    if dtype in _FLOATS:
        return KVCache(k, v)
    return KVCache(k, v, *(torch.ones(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))


def _cache(cache, device=None):
    """Check a cache; -> (k, pointers, strides) as the kernels take them."""
    k, v, ks, vs = cache
    _tensor(k, "cache.k", 4, _TYPE, device)
    dev = k.device
    _tensor(v, "cache.v", 4, (k.dtype,), dev)
    if v.shape != k.shape:
        raise ValueError(f"cache.k {tuple(k.shape)} and cache.v {tuple(v.shape)} must have one shape")
    if k.shape[0] * k.shape[1] >= 1 << 31:
        raise ValueError("a cache has at most 2^31 - 1 slots")
    st = k.stride()[:3] + v.stride()[:3]
    if k.dtype in _FLOATS:
        if ks is not None or vs is not None:
            raise ValueError(f"a {k.dtype} cache has no scales")
        return k, (k.data_ptr(), v.data_ptr(), 0, 0), st + (0,) * 6
    for s, name in ((ks, "cache.k_scales"), (vs, "cache.v_scales")):
        if s is None:
            raise ValueError(f"{name}: an 8-bit cache has scales")
        if not isinstance(s, torch.Tensor) or s.device != dev or s.dtype != torch.float32 or s.shape != k.shape[:3]:
            raise ValueError(f"{name} must be an fp32 tensor of {tuple(k.shape[:3])} on {dev}")
    return k, (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()), st + ks.stride() + vs.stride()


def _slots(slots, device):
    _tensor(slots, "slots", 1, _INDEX, device, contiguous=True)
    return slots.shape[0]


def kv_cache_write(cache: KVCache, k, v, slots) -> KVCache:
    """Write rows ``k``, ``v`` [T, heads, dim] (fp32, fp16 or bf16, any strides
    but a contiguous last dimension) at ``slots`` [T] (int32 or int64; a slot is
    page * page size + offset), and return the cache.

    An 8-bit cache is quantised on the way, with one fp32 scale for each head of
    a row, and a value is code * scale: float8_e4m3fn under the least power of
    two that brings the head's largest value to 448 or less (so scaling rounds
    nothing), int8 under the largest value / 127.  A head that holds an infinity
    or a NaN reads back as NaN in 8 bits.  A row whose slot is negative or behind
    the cache is left out (padding).  Slots must not name the same place twice:
    which row's values it would hold is not defined.
    """
    c, ptrs, cst = _cache(cache)
    dev = c.device
    pages, page, heads, dim = c.shape
    _tensor(k, "k", 3, _FLOATS, dev)
    _tensor(v, "v", 3, (k.dtype,), dev)
    T = _slots(slots, dev)
    for x, name in ((k, "k"), (v, "v")):
        if x.shape != (T, heads, dim):
            raise ValueError(f"{name} must be {(T, heads, dim)}, got {tuple(x.shape)}")
    if dim > 512:
        raise ValueError(f"dim must be at most 512, got {dim}")
    if T:
        _launch(c, _k().kv_cache_write, (k.data_ptr(), v.data_ptr()), k.stride()[:2] + v.stride()[:2], _TYPE[k.dtype], ptrs,
                cst, _TYPE[c.dtype], pages, page, slots.data_ptr(), _INDEX[slots.dtype], T, heads, dim)
    return cache


def kv_cache_read(cache: KVCache, slots, dtype=None) -> Tuple:
    """The rows at ``slots`` [T] of a cache as (k, v) [T, heads, dim] in
    ``dtype`` (fp32, fp16 or bf16; the cache's own, or bf16 for an 8-bit one).
    A slot that is negative or behind the cache gives zeros."""
    c, ptrs, cst = _cache(cache)
    pages, page, heads, dim = c.shape
    dtype = dtype or (c.dtype if c.dtype in _FLOATS else torch.bfloat16)
    if dtype not in _FLOATS:
        raise TypeError(f"dtype must be one of {[str(d) for d in _FLOATS]}, got {dtype}")
    T = _slots(slots, c.device)
    if dim > 512:
        raise ValueError(f"dim must be at most 512, got {dim}")
    k, v = (torch.empty((T, heads, dim), dtype=dtype, device=c.device) for _ in range(2))
    if T:
        _launch(c, _k().kv_cache_read, (k.data_ptr(), v.data_ptr()), k.stride()[:2] + v.stride()[:2], _TYPE[dtype], ptrs, cst,
                _TYPE[c.dtype], pages, page, slots.data_ptr(), _INDEX[slots.dtype], T, heads, dim)
    return k, v


# ------------------------------------------------------------ CPU references
def qk_norm_rope_ref(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False):
    """64-bit reference of :func:`qk_norm_rope` on any device."""
    angle = positions.double()[:, None] * inv_freq.double()[None]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    n = inv_freq.shape[0]
    outs = []
    for x, w in ((q, q_weight), (k, k_weight)):
        x = x.double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        if w is not None:
            x = x * w.double()
        y = x.clone()
        ia = slice(0, 2 * n, 2) if interleaved else slice(0, n)
        ib = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
        y[..., ia] = x[..., ia] * cos - x[..., ib] * sin
        y[..., ib] = x[..., ib] * cos + x[..., ia] * sin
        outs.append(y)
    return tuple(outs)


def kv_quantise_ref(x, dtype):
    """(codes, scales) of rows in an 8-bit cache: [..., dim] -> [..., dim] and [...]."""
    x = x.float()
    top = x.abs().amax(-1)
    if dtype == torch.float8_e4m3fn:
        m, e = torch.frexp(torch.nan_to_num(top))
        k = torch.where(m <= 0.875, e - 9, e - 8).clamp(-120, 120).int()
        scale = ((k + 127) << 23).view(torch.float32)
    else:
        scale = (top * (1.0 / 127.0)).clamp_min(2.0 ** -120)
    scale = torch.where(top > 0, scale, torch.ones_like(scale))
    scale = torch.where(torch.isfinite(top), scale, torch.full_like(scale, float("nan")))
    y = x / scale[..., None]
    if dtype == torch.float8_e4m3fn:
        return y.to(dtype), scale
    return torch.nan_to_num(y).round().clamp(-127, 127).to(torch.int8), scale
