"""Operators of one step of a served token model.

A decoder's attention block between its projections, as a GPU component calls
it, eagerly or through a graph that it captures::

    qkv = ops.lora_add(F.linear(x, w_qkv), x, A, B, tenant)     # adapters of many tenants
    q, k, v = qkv.view(T, -1, D).split((Hq, Hk, Hk), 1)
    q, k = ops.qk_norm_rope(q, k, q_norm, k_norm, positions, inv_freq)
    ops.kv_cache_write(cache, k, v, slots)                        # 16 or 8 bits
    y = ops.paged_attention(q, cache, page_table, lengths)        # one new token per request

Every op launches hand-written HIP kernels on the current stream of its
tensors' device, allocates only its outputs and workspace (from torch's
allocator, so a captured graph keeps its own) and never synchronises: lengths,
page tables, slots and adapter ids are read on the GPU only.  What the host can
see (shapes, types, strides, devices, tensors without memory, as tracers use
them) is checked and refused with ``ValueError`` / ``TypeError``; indices that
point outside a cache or a table are left out by the kernels as each op says.
The ops are forward only (``RuntimeError`` where a gradient or a tangent would
be lost).

A captured step pads its batch with rows whose slot is -1 (nothing is written)
and whose length is 0.  :class:`~seldon_core_amd.models.graphed.GraphedModule`
pads with zeros and runs a module on zeros before it captures it, which is right
for modules that keep nothing; in it ``kv_cache_write`` raises, and a module
that writes a cache is served eagerly.

Kernel sources: csrc/kernels/{rope,kv_cache,paged_attention,lora}.hip.
"""
from __future__ import annotations

import contextlib
import functools
import threading
from typing import NamedTuple, Optional, Tuple

from .._native import native

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None

if torch is not None:
    import torch.autograd.forward_ad as _forward_ad

    _TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3, torch.int8: 4}
    _FLOATS = (torch.float32, torch.float16, torch.bfloat16)
    _INDEX = {torch.int32: 0, torch.int64: 1}
    _NEGATED = (torch.float32, torch.float16)  # types that views of complex numbers have
    _Tensor = torch.Tensor
    _increment_version = torch.autograd.graph.increment_version

_kernels = None


def _k():
    global _kernels
    if _kernels is None:
        _kernels = native().kernels
    return _kernels


# A call's checks are most of its host time, which bounds the small ones (about 0.1 us for each question asked of a tensor):
# nothing is asked twice, and rare properties only where the type can have them.
def _tensor(t, name, dim, dtypes, device=None, contiguous=False):
    """Refuse what the kernels do not take; ``contiguous``: every stride, else only the last.  ``device``: a GPU."""
    if not isinstance(t, _Tensor) or (not t.is_cuda if device is None else t.device != device):
        if isinstance(t, _Tensor) and t.is_cuda:
            raise ValueError(f"{name} is on {t.device}, not {device}")
        raise ValueError(f"{name} must be a GPU tensor")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, got {tuple(t.shape)}")
    dtype = t.dtype
    if dtype not in dtypes:
        raise TypeError(f"{name} must be one of {[str(d) for d in dtypes]}, got {dtype}")
    if contiguous:
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    elif t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    if t.requires_grad or _forward_ad._current_level >= 0 or dtype in _NEGATED and t.is_neg():
        _as_stored(t, name)
    return t


def _as_stored(t, name):
    """Refuse a tensor that is more than its memory says: a sign put off, a gradient or a tangent (forward mode)."""
    if t.is_neg():
        raise ValueError(f"{name} is a view whose sign is put off (the imaginary part of a conjugate); use {name}.resolve_neg()")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient; this operator is forward only (use torch.no_grad())")
    # a dual tensor does not require a gradient; outside of a dual level (-1) there are none
    if _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{name} has a tangent; this operator has no derivative (use forward_ad.unpack_dual(x).primal)")


if torch is not None and hasattr(torch._C, "_cuda_getCurrentRawStream") and hasattr(torch._C, "_cuda_getDevice"):
    _stream_of = torch._C._cuda_getCurrentRawStream  # 1.7 us less a call than the Stream object
    _current_device = torch._C._cuda_getDevice  # the public one asks first whether there is a GPU
else:  # pragma: no cover
    def _stream_of(index):
        return torch.cuda.current_stream(index).cuda_stream

    def _current_device():
        return torch.cuda.current_device()


def _launch(t, fn, *args):
    """fn(*args, stream) on the current stream of t's device."""
    index = t.device.index
    if _current_device() == index:
        fn(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            fn(*args, _stream_of(index))


def _optional(t, name):
    """The address of a tensor that may be None: 0 for None only (the kernels refuse a null pointer elsewhere)."""
    return 0 if t is None else t.data_ptr() or _no_memory(t, name)


def _no_memory(t, name):
    if t.numel():
        raise ValueError(f"{name} has no memory")
    return 0


def _written(t, name):
    """Refuse a tensor to write that holds an element twice (an expanded one)."""
    if 0 in t.stride() and any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
        raise ValueError(f"{name} holds elements more than once (it is expanded), and is written")


def _in_place(out, t):
    return out is t or out.data_ptr() == t.data_ptr() and out.stride() == t.stride()


def _apart(out, t, name, other):
    """Refuse an output over an input, as far as the host can tell: a common start, or ranges of two contiguous tensors that meet."""
    a, b = out.data_ptr(), t.data_ptr()
    if a < b + t.nbytes and b < a + out.nbytes and (a == b or out.is_contiguous() and t.is_contiguous()):
        raise ValueError(f"{name} lies over {other}")


def _changed(tensors):
    """Tell autograd that tensors of the caller's were written over: a backward pass may have kept them, also where the writing is
    under no_grad or in inference mode."""
    _increment_version(tensors)


def _new(t):
    """An uninitialised contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


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
    inputs themselves (other overlaps are not allowed).  Sums of squares are
    fp32: heads with values beyond about 10^18 overflow them and give zeros.
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
        oq, ok = _new(q), _new(k)
    else:
        oq, ok = out
        for o, x, name in ((oq, q, "out[0]"), (ok, k, "out[1]")):
            _tensor(o, name, 3, (dt,), dev)
            if o.shape != x.shape:
                raise ValueError(f"{name} must be {tuple(x.shape)}, got {tuple(o.shape)}")
            _written(o, name)
            if not _in_place(o, x):
                _apart(o, x, name, "its input")
        _apart(oq, k, "out[0]", "k")
        _apart(ok, q, "out[1]", "q")
        _apart(oq, ok, "out[0]", "out[1]")
    if T and Hq + Hk:
        _launch(q, _k().qk_norm_rope, q.data_ptr(), k.data_ptr(), oq.data_ptr(), ok.data_ptr(),
                _optional(q_weight, "q_weight"), _optional(k_weight, "k_weight"), bool(wf32),
                q.stride()[:2] + k.stride()[:2] + oq.stride()[:2] + ok.stride()[:2], T, Hq, Hk, D, _TYPE[dt],
                positions.data_ptr(), _INDEX[positions.dtype], inv_freq.data_ptr(), inv_freq.dtype == torch.float64,
                inv_freq.shape[0], interleaved, eps)
        if out is not None:
            _changed((oq, ok))
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
    float8_e4m3fn or int8 for one that is quantised as it is written.

    A page keeps the rows of a head together (the tensors are transposed views):
    attention reads one head at a time, and where rows are not whole 128-byte
    lines it would otherwise fetch its neighbours' too (36 requests of 3000
    tokens, 12 heads, kernels alone: 44 against 67 us at e4m3 and dim 64, 123
    against 133 at bf16 and dim 128).

    Any dim up to 512 in any of the types can be written and read.
    :func:`paged_attention` takes bf16, fp16 and 8-bit caches whose dim is at
    most 256 and a multiple of 8 (of 16 in 8 bits); fp32 caches and other dims
    are for attention of the caller's own over rows read back.  A dim that is no
    multiple of 8 is written and read value by value, which is slower.
    """
    dtype = dtype or torch.bfloat16
    if dtype not in _TYPE:
        raise TypeError(f"dtype must be one of {[str(d) for d in _TYPE]}, got {dtype}")
    if min(pages, page_size, heads, dim) < 1:
        raise ValueError("pages, page_size, heads and dim must be positive")
    shape = (pages, heads, page_size, dim)
    k, v = (torch.zeros(shape, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))
    if dtype in _FLOATS:
        return KVCache(k, v)
    return KVCache(k, v, *(torch.ones(shape[:3], dtype=torch.float32, device=device).transpose(1, 2) for _ in range(2)))


def _cache(cache, device=None):
    """Check a cache; -> (k, its shape, pointers, strides) as the kernels take them."""
    k, v, ks, vs = cache
    _tensor(k, "cache.k", 4, _TYPE, device)
    dev = k.device
    _tensor(v, "cache.v", 4, (k.dtype,), dev)
    shape = k.shape
    if v.shape != shape:
        raise ValueError(f"cache.k {tuple(shape)} and cache.v {tuple(v.shape)} must have one shape")
    if shape[0] * shape[1] >= 1 << 31:
        raise ValueError("a cache has at most 2^31 - 1 slots")
    st = k.stride()[:3] + v.stride()[:3]
    if k.dtype in _FLOATS:
        if ks is not None or vs is not None:
            raise ValueError(f"a {k.dtype} cache has no scales")
        return k, shape, (k.data_ptr(), v.data_ptr(), 0, 0), st + (1,) * 6
    rows = shape[:3]
    for s, name in ((ks, "cache.k_scales"), (vs, "cache.v_scales")):
        if s is None:
            raise ValueError(f"{name}: an 8-bit cache has scales")
        if not isinstance(s, _Tensor) or s.shape != rows or s.dtype != torch.float32 or s.device != dev:
            raise ValueError(f"{name} must be an fp32 tensor of {tuple(rows)} on {dev}")
        if s.requires_grad or _forward_ad._current_level >= 0 or s.is_neg():
            _as_stored(s, name)
    return k, shape, (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()), st + ks.stride() + vs.stride()


class _Rehearsal(threading.local):
    why = None


_rehearsal = _Rehearsal()


@contextlib.contextmanager
def no_cache_writes(why: str):
    """In this thread :func:`kv_cache_write` raises: for callers that run a module on rows that are no request's."""
    before, _rehearsal.why = _rehearsal.why, why
    try:
        yield
    finally:
        _rehearsal.why = before


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
    it would hold parts of several rows, under the scale of one of them; nor may a
    row be read that is written (``k`` and ``v`` may be other rows of the cache).
    """
    if _rehearsal.why:
        raise RuntimeError(f"the cache is not written: {_rehearsal.why}")
    c, (pages, page, heads, dim), ptrs, cst = _cache(cache)
    dev = c.device
    _tensor(k, "k", 3, _FLOATS, dev)
    _tensor(v, "v", 3, (k.dtype,), dev)
    T = _slots(slots, dev)
    shape = (T, heads, dim)
    for x, name in ((k, "k"), (v, "v")):
        if x.shape != shape:
            raise ValueError(f"{name} must be {shape}, got {tuple(x.shape)}")
    if dim > 512:
        raise ValueError(f"dim must be at most 512, got {dim}")
    if 0 in cst:
        for t, name in zip(cache, ("cache.k", "cache.v", "cache.k_scales", "cache.v_scales")):
            if t is not None:
                _written(t, name)
    if T:
        _launch(c, _k().kv_cache_write, (k.data_ptr(), v.data_ptr()), k.stride()[:2] + v.stride()[:2], _TYPE[k.dtype], ptrs,
                cst, _TYPE[c.dtype], pages, page, slots.data_ptr(), _INDEX[slots.dtype], T, heads, dim)
        _changed(cache[:2] if c.dtype in _FLOATS else cache)
    return cache


def kv_cache_read(cache: KVCache, slots, dtype=None) -> Tuple:
    """The rows at ``slots`` [T] of a cache as (k, v) [T, heads, dim] in
    ``dtype`` (fp32, fp16 or bf16; the cache's own, or bf16 for an 8-bit one).
    A slot that is negative or behind the cache gives zeros."""
    c, (pages, page, heads, dim), ptrs, cst = _cache(cache)
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


# --------------------------------------------------------------- attention
_workspace = None


def _attention_workspace(*sizes):
    """fp32 numbers of workspace for (batch, kv heads, group, dim, 8 bits, tokens, window)."""
    global _workspace
    if _workspace is None:
        _workspace = functools.lru_cache(maxsize=1024)(_k().paged_attention_workspace)
    return _workspace(*sizes)


def paged_attention(q, cache: KVCache, page_table, lengths, *, scale: Optional[float] = None, window: int = 0,
                    return_lse: bool = False, out=None):
    """Attention of one new token per request over its tokens in a paged cache.

    ``q`` [B, Hq, D] (fp16 or bf16, any strides but a contiguous last
    dimension); the ``cache`` is of q's type, float8_e4m3fn or int8, and query
    head h reads its head h // (Hq / H).  ``page_table`` [B, W] (int32 only; rows
    may be strided) names each request's pages in order, ``lengths`` [B] (int32
    only) how many tokens it has, its new one among them: that one sees all of
    them, or the last ``window``.  ``scale`` is D ** -0.5 unless given.

    D is at most 256 and a row of the cache a multiple of 16 bytes (D a multiple
    of 8, of 16 with 8 bits), starting at one.  A length beyond the table counts
    as the table's end, a negative one as 0; tokens on a page outside the cache
    are left out, and what the cache holds where nothing is seen (anything, NaN
    too) does not matter.  A request that sees nothing, or nothing but scores of
    -inf, gets zeros.  Where a value that is seen is NaN, so is its dimension;
    where one is infinite its dimension is infinite or NaN, never finite (a
    weight enters as the sum of two 16-bit numbers, of which one can be 0 or
    negative).  In 8 bits the head's scale is NaN then, and so are all of its
    dimensions.  Sums are fp32 and divided by the softmax's total at the end, so
    values beyond about 10^30 can overflow.

    Returns [B, Hq, D] in q's type (``out`` if given: contiguous, not
    overlapping q), with ``return_lse`` also the natural logsumexp of its scores
    [B, Hq] in fp32, -inf where nothing is seen.
    """
    _tensor(q, "q", 3, (torch.bfloat16, torch.float16))
    dev = q.device
    c, (pages, page, H, dim), ptrs, cst = _cache(cache, dev)
    B, Hq, D = q.shape
    if c.dtype.itemsize != 1 and c.dtype != q.dtype:
        raise TypeError(f"a cache of {c.dtype} does not go with queries of {q.dtype}")
    if dim != D or not H or not Hq or Hq % H:
        raise ValueError(f"queries {tuple(q.shape)} do not go with a cache of {H} heads of {dim}")
    if D > 256 or D * c.dtype.itemsize % 16:
        raise ValueError(f"dim must be at most 256 and fill multiples of 16 bytes in the cache, got {D} of {c.dtype}")
    _tensor(page_table, "page_table", 2, (torch.int32,), dev)
    _tensor(lengths, "lengths", 1, (torch.int32,), dev, contiguous=True)
    W = page_table.shape[1]
    if page_table.shape[0] != B or lengths.shape[0] != B:
        raise ValueError(f"page_table {tuple(page_table.shape)} and lengths {tuple(lengths.shape)} must have {B} rows")
    if not 1 <= W * page <= 1 << 30:
        raise ValueError(f"page_table holds {W * page} tokens for a request: at least 1, at most 2^30")
    if window < 0:
        raise ValueError(f"window must not be negative, got {window}")
    window = min(window, W * page)  # a larger one sees all, and may be no 32-bit number
    given = out is not None
    if not given:
        out = _new(q)
    else:
        _tensor(out, "out", 3, (q.dtype,), dev, contiguous=True)
        if out.shape != q.shape:
            raise ValueError(f"out must be {tuple(q.shape)}, got {tuple(out.shape)}")
        _apart(out, q, "out", "q")
    lse = torch.empty((B, Hq), dtype=torch.float32, device=dev) if return_lse else None
    if B:
        n = _attention_workspace(B, H, Hq // H, D, c.dtype.itemsize == 1, W * page, window)
        ws = torch.empty(n, dtype=torch.float32, device=dev)
        _launch(q, _k().paged_attention, q.data_ptr(), q.stride(0), q.stride(1), _TYPE[q.dtype], ptrs, cst, _TYPE[c.dtype],
                pages, page, page_table.data_ptr(), page_table.stride(0), W, lengths.data_ptr(), B, H, Hq // H, D, window,
                D ** -0.5 if scale is None else scale, out.data_ptr(), 0 if lse is None else lse.data_ptr(), ws.data_ptr(), n)
        if given:
            _changed((out,))
    return (out, lse) if return_lse else out


# ---------------------------------------------------------------- adapters
_lora_workspace = None


def lora_add(y, x, A, B, adapters, scales=None, out=None):
    """``y + scales[a] * (x @ A[a].T) @ B[a].T`` with the adapter ``a`` of each
    row: low-rank adapters of many requests at once beside the projection whose
    output ``y`` is.

    ``x`` [T, K] and ``y`` [T, M] (fp32, fp16 or bf16, all of one type; rows may
    be strided, such as a part of a fused projection); ``A`` [N, r, K] and ``B``
    [N, M, r], contiguous, r at most 128 (pad a smaller rank with zeros);
    ``adapters`` [T] int32 or int64; ``scales`` [N] fp32.  A row whose adapter is
    negative or behind the last keeps y.  Rows may come in any order; many rows
    are fastest where those of one adapter lie together (of up to 2000 adapters
    they are brought together first, of more they are not).

    Sums are fp32, with one rounding at the end.  Where a weight of B is infinite
    the result is: with fp32 tensors the infinity (or, next to a 0, the NaN) that
    the formula has; with 16-bit ones infinite or NaN, since ``A x`` enters the
    second product as the sum of two 16-bit numbers.  Returns a new tensor, or
    ``out``, which may be ``y`` itself (other overlaps are not allowed).
    """
    global _lora_workspace
    _tensor(y, "y", 2, _FLOATS)
    dev, dt = y.device, y.dtype
    _tensor(x, "x", 2, (dt,), dev)
    _tensor(A, "A", 3, (dt,), dev, contiguous=True)
    _tensor(B, "B", 3, (dt,), dev, contiguous=True)
    T, M = y.shape
    N, r, K = A.shape
    if x.shape != (T, K) or B.shape != (N, M, r):
        raise ValueError(f"x {tuple(x.shape)}, y {tuple(y.shape)}, A {tuple(A.shape)} and B {tuple(B.shape)} do not go together")
    if not 1 <= r <= 128 or not 1 <= K <= 1 << 24 or M > 1 << 24 or not N:
        raise ValueError(f"rank must be 1 to 128 and there must be an adapter, got A {tuple(A.shape)}")
    _tensor(adapters, "adapters", 1, _INDEX, dev, contiguous=True)
    if adapters.shape[0] != T:
        raise ValueError(f"adapters must have {T} values, got {adapters.shape[0]}")
    if scales is not None:
        _tensor(scales, "scales", 1, (torch.float32,), dev, contiguous=True)
        if scales.shape[0] != N:
            raise ValueError(f"scales must have {N} values, got {scales.shape[0]}")
    given = out is not None
    if not given:
        out = _new(y)
    else:
        _tensor(out, "out", 2, (dt,), dev)
        if out.shape != y.shape:
            raise ValueError(f"out must be {tuple(y.shape)}, got {tuple(out.shape)}")
        _written(out, "out")
        if not _in_place(out, y):
            _apart(out, y, "out", "y")
        _apart(out, x, "out", "x")
    if T and M:
        if _lora_workspace is None:
            _lora_workspace = functools.lru_cache(maxsize=1024)(_k().lora_workspace)
        n = _lora_workspace(T, K, r, N)
        ws = torch.empty(n, dtype=torch.float32, device=dev)
        _launch(y, _k().lora_add, y.data_ptr(), y.stride(0), x.data_ptr(), x.stride(0), out.data_ptr(), out.stride(0),
                A.data_ptr(), B.data_ptr(), adapters.data_ptr(), _INDEX[adapters.dtype],
                _optional(scales, "scales"), T, K, M, r, N, _TYPE[dt], ws.data_ptr(), n)
        if given:
            _changed((out,))
    return out


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


def paged_attention_ref(q, cache, page_table, lengths, scale=None, window=0):
    """64-bit reference of :func:`paged_attention` -> (out, lse, sum of |weight * value|)."""
    B, Hq, D = q.shape
    pages, page, H, _ = cache.k.shape
    g = Hq // H
    scale = D ** -0.5 if scale is None else scale
    out, mag = (torch.zeros((B, Hq, D), dtype=torch.float64) for _ in range(2))
    lse = torch.full((B, Hq), float("-inf"), dtype=torch.float64)

    def rows(x, s, p, at):
        y = x[p, at].float().double() if s is not None else x[p, at].double()
        return y if s is None else y * s[p, at].double()[..., None]

    for b in range(B):
        n = min(max(int(lengths[b]), 0), page_table.shape[1] * page)
        t = torch.arange(max(0, n - window) if window else 0, n)
        p = page_table[b][t // page].long()
        keep = (p >= 0) & (p < pages)
        t, p = t[keep], p[keep]
        if not len(t):
            continue
        k, v = rows(cache.k, cache.k_scales, p, t % page), rows(cache.v, cache.v_scales, p, t % page)
        for h in range(Hq):
            s = k[:, h // g] @ q[b, h].double() * scale
            lse[b, h] = torch.logsumexp(s, 0)
            w = torch.softmax(s, 0)
            out[b, h], mag[b, h] = w @ v[:, h // g], w @ v[:, h // g].abs()
    return out, lse, mag


def lora_add_ref(y, x, A, B, adapters, scales=None):
    """64-bit reference of :func:`lora_add` -> (out, sum of |x||A||B| as a measure of its rounding)."""
    out = y.double().clone()
    mag = torch.zeros_like(out)
    for a in range(A.shape[0]):
        rows = (adapters == a).nonzero()[:, 0]
        s = 1.0 if scales is None else scales[a].double()
        Aa, Ba, xa = A[a].double(), B[a].double(), x[rows].double()
        out[rows] += s * ((xa @ Aa.T) @ Ba.T)
        mag[rows] = abs(s) * ((xa.abs() @ Aa.abs().T) @ Ba.abs().T)
    return out, mag
