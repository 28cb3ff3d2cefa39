"""Serving operators on CUDA tensors: pages for new tokens, an 8-bit paged KV cache and the attention over it, sampling.

One step of a serving loop, all on the current stream of the tensors' device and with no host read in between::

    step = reserve_pages(table, kv_len, new_tokens, ring, free_state, page_size=16, max_tokens=n)
    append_kv8(k, v, step.slots, k_cache, v_cache, k_scale, v_scale)
    out = attend_kv8(q, k_cache, v_cache, k_scale, v_scale, table, step.kv_len, q_start=step.q_start, max_q=m)
    token, logprob = sample_tokens(logits, u, temperature=t, top_p=p)

They call the C entry points ``ptowsp_cuda_reserve_pages``, ``_kv8_append``, ``_kv8_attention`` and ``_sample_tokens``
(``include/ptowsp_cuda.h`` has their definitions).  Arguments that a call does not take raise ``TypeError`` or
``ValueError`` here, or :class:`~pto_wsp_b200.runtime.PtoWspCudaError` with the library's status.  What only the device
sees (a page id outside the cache, a request without room) is or'ed into the ``status`` tensor, an int32 that the caller
zeroes; :func:`check_status` reads it and raises.  The calls allocate their results (and the attention its workspace)
with torch's allocator on the current stream, and keep nothing.  They have no gradient: inputs that require one are
refused (``ValueError``) unless gradients are off, as under ``torch.no_grad()``.
"""

from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple

import torch

from .runtime import PTOWSP_OK, PtoWspCudaError, load_library

_P, _I64, _I32, _F32 = C.c_void_p, C.c_int64, C.c_int32, C.c_float
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_FORMATS = {torch.float8_e4m3fn: 0, torch.int8: 1}

PAGE, LENGTH, REFUSED, RING, TIMEOUT = 1, 2, 4, 8, 16  # bits of a status tensor
_STATUS_TEXT = {PAGE: "a page id or slot outside the cache", LENGTH: "a length that is negative or beyond its table",
                REFUSED: "a request's new tokens found no room", RING: "the free-page ring is inconsistent",
                TIMEOUT: "a bounded wait gave up"}


class _Reserve(C.Structure):
    _fields_ = [("page_table", _P), ("table_stride", _I64), ("max_pages", _I32), ("page_size", _I32),
                ("requests", _I32), ("reserved0", _I32), ("kv_len", _P), ("new_tokens", _P), ("free_ring", _P),
                ("ring_size", _I64), ("free_state", _P), ("slots", _P), ("positions", _P), ("max_tokens", _I64),
                ("q_start", _P), ("kv_len_out", _P), ("free_state_out", _P), ("granted", _P), ("status", _P)]


class _Cache(C.Structure):
    _fields_ = [("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P), ("k_page_stride", _I64),
                ("k_token_stride", _I64), ("k_head_stride", _I64), ("v_page_stride", _I64), ("v_token_stride", _I64),
                ("v_head_stride", _I64), ("num_pages", _I64), ("page_size", _I32), ("num_kv_heads", _I32),
                ("head_dim", _I32), ("format", _I32)]


class _Append(C.Structure):
    _fields_ = [("k", _P), ("v", _P), ("k_token_stride", _I64), ("k_head_stride", _I64), ("v_token_stride", _I64),
                ("v_head_stride", _I64), ("slots", _P), ("tokens", _I64), ("dtype", _I32), ("reserved0", _I32),
                ("status", _P)]


class _Attention(C.Structure):
    _fields_ = [("q", _P), ("out", _P), ("lse", _P), ("q_token_stride", _I64), ("q_head_stride", _I64),
                ("out_token_stride", _I64), ("out_head_stride", _I64), ("page_table", _P), ("table_stride", _I64),
                ("kv_len", _P), ("q_start", _P), ("tokens", _I64), ("max_pages", _I32), ("requests", _I32),
                ("num_heads", _I32), ("max_q", _I32), ("window", _I32), ("dtype", _I32), ("scale", _F32),
                ("reserved0", _I32), ("workspace", _P), ("workspace_bytes", C.c_size_t), ("status", _P)]


class _Sample(C.Structure):
    _fields_ = [("logits", _P), ("row_stride", _I64), ("rows", _I32), ("vocab", _I32), ("dtype", _I32),
                ("reserved0", _I32), ("u", _P), ("temperature", _P), ("top_k", _P), ("top_p", _P), ("min_p", _P),
                ("token", _P), ("logprob", _P)]


def _packer(cls):
    """The struct's C layout as a bytes packer: filling a ctypes structure field by field takes twice as long."""
    codes = {_P: "P", _I64: "q", _I32: "i", _F32: "f", C.c_size_t: "N"}
    fmt = struct.Struct("@" + "".join(codes[t] for _, t in cls._fields_))
    assert fmt.size == C.sizeof(cls)
    return fmt.pack


_pack_reserve, _pack_cache, _pack_append, _pack_attention, _pack_sample = map(
    _packer, (_Reserve, _Cache, _Append, _Attention, _Sample))
_lib = None


def _library():
    global _lib
    if _lib is None:
        lib = load_library()
        for name, args in (("reserve_pages", 1), ("kv8_append", 2), ("kv8_attention", 2), ("sample_tokens", 1)):
            fn = getattr(lib, "ptowsp_cuda_" + name)
            fn.argtypes, fn.restype = [_P] * (args + 1), C.c_int
        lib.ptowsp_cuda_kv8_attention_workspace.argtypes = [_P, _P]
        lib.ptowsp_cuda_kv8_attention_workspace.restype = C.c_size_t
        _lib = lib
    return _lib


def _call(fn, index, *structs):
    """Call a C entry on device `index` and its current stream (read as torch.cuda.current_stream reads it)."""
    if index == torch._C._cuda_getDevice():
        rc = fn(*structs, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*structs, torch._C._cuda_getCurrentRawStream(index))
    if rc != PTOWSP_OK:
        raise PtoWspCudaError(rc, (_library().ptowsp_cuda_last_error() or b"").decode())


def _need(cond, text):
    if not cond:
        raise ValueError(text)


def _no_gradient():
    if torch.is_grad_enabled():
        raise ValueError("the serving operators have no gradient: call them under torch.no_grad(), or detach the inputs")


def _cuda_index(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _vector(t, name, dtype, n, index):
    """A contiguous 1-D tensor of n elements, as its address; 0 for None."""
    if t is None:
        return 0
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
    if t.shape != (n,) or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"{name} must be contiguous, of {n} elements, on cuda:{index} (got {tuple(t.shape)} on {t.device})")
    return t.data_ptr()


def _table(t, requests, index):
    if t.dtype is not torch.int32:
        raise TypeError(f"page_table must be torch.int32 (got {t.dtype})")
    shape = t.shape
    if len(shape) != 2 or shape[0] != requests or t.get_device() != index or (shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"page_table must be [{requests}, max_pages] on cuda:{index}, its rows contiguous")
    return t.data_ptr(), t.stride(0) if requests > 1 else shape[1], shape[1]


def check_status(status: torch.Tensor) -> None:
    """Read a status tensor (waiting for the work that writes it), zero it, and raise if a bit was set."""
    bits = int(status.item())
    if bits:
        status.zero_()
        raise PtoWspCudaError(5, "; ".join(text for bit, text in _STATUS_TEXT.items() if bits & bit))


class PageStep(NamedTuple):
    """What :func:`reserve_pages` gives."""

    slots: torch.Tensor       # int64 [max_tokens]: page * page_size + offset of each new token, -1: none
    positions: torch.Tensor   # int32 [max_tokens]: its position in its request, -1: none
    q_start: torch.Tensor     # int32 [requests + 1]: prefix sums of the new tokens
    kv_len: torch.Tensor      # int32 [requests]: lengths with the new tokens
    free_state: torch.Tensor  # int64 [2]: head and tail of the free-page ring
    granted: torch.Tensor     # bool [requests]


def reserve_pages(page_table, kv_len, new_tokens, free_ring, free_state, *, page_size: int, max_tokens: int,
                  status=None) -> PageStep:
    """Give pages to the new tokens of each request and take back those of requests that ended (``new_tokens`` < 0).

    ``page_table`` int32 [requests, max_pages] and ``free_ring`` int32 [n] are updated in place; ``kv_len`` and
    ``new_tokens`` are int32 [requests], ``free_state`` int64 [2] (head, tail: the ring holds the free page ids at
    head .. tail - 1 modulo n).  ``max_tokens``: length of the token list, at least the sum of the new tokens.
    A request that finds no room is refused whole: its length stays and its slots are -1."""
    index = _cuda_index(page_table, "page_table")
    i32, i64 = torch.int32, torch.int64
    requests, cap = kv_len.shape[0], free_ring.shape[0]
    table, stride, max_pages = _table(page_table, requests, index)
    _need(max_tokens >= 0, "max_tokens must not be negative")
    len_in, state_in = _vector(kv_len, "kv_len", i32, requests, index), _vector(free_state, "free_state", i64, 2, index)
    len_out, state_out = torch.empty_like(kv_len), torch.empty_like(free_state)
    q_start, positions, slots = kv_len.new_empty(requests + 1), kv_len.new_empty(max_tokens), free_state.new_empty(max_tokens)
    granted = torch.empty_like(kv_len, dtype=torch.bool)
    _call(_library().ptowsp_cuda_reserve_pages, index, _pack_reserve(
        table, stride, max_pages, page_size, requests, 0, len_in,
        _vector(new_tokens, "new_tokens", i32, requests, index), _vector(free_ring, "free_ring", i32, cap, index), cap,
        state_in, slots.data_ptr(), positions.data_ptr(), max_tokens, q_start.data_ptr(), len_out.data_ptr(),
        state_out.data_ptr(), granted.data_ptr(), _vector(status, "status", i32, 1, index)))
    return PageStep(slots, positions, q_start, len_out, state_out, granted)


def _cache(k_cache, v_cache, k_scale, v_scale):
    """Checks a cache; its device, the packed struct, heads and head_dim."""
    index = _cuda_index(k_cache, "k_cache")
    fmt = _FORMATS.get(k_cache.dtype)
    if fmt is None or v_cache.dtype is not k_cache.dtype:
        raise TypeError(f"k_cache and v_cache must both be float8_e4m3fn or int8 (got {k_cache.dtype}, {v_cache.dtype})")
    shape, ks, vs = k_cache.shape, k_cache.stride(), v_cache.stride()
    if len(shape) != 4 or v_cache.shape != shape or ks[3] != 1 or vs[3] != 1 or v_cache.get_device() != index:
        raise ValueError(f"k_cache and v_cache must be [pages, page_size, heads, head_dim] on cuda:{index}, the last "
                         f"dimension contiguous (got {tuple(shape)}, {tuple(v_cache.shape)})")
    pages, page, heads, dim = shape
    for t in (k_scale, v_scale):
        if t.dtype is not torch.float32:
            raise TypeError(f"k_scale and v_scale must be torch.float32 (got {t.dtype})")
        if t.shape != (pages, heads) or not t.is_contiguous() or t.get_device() != index:
            raise ValueError(f"k_scale and v_scale must be contiguous [{pages}, {heads}] on cuda:{index}")
    return index, _pack_cache(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), ks[0],
                              ks[1], ks[2], vs[0], vs[1], vs[2], pages, page, heads, dim, fmt), heads, dim


def append_kv8(k, v, slots, k_cache, v_cache, k_scale, v_scale, *, status=None) -> None:
    """Write the rows ``k``, ``v`` [tokens, heads, head_dim] (float32, float16 or bfloat16) into the cache at ``slots``
    (int64 [tokens], -1: skip; those of one page next to each other and ascending, none twice and no -1 between them).

    The cache, codes [pages, page_size, heads, head_dim] in float8_e4m3fn or int8 with any page, token and head order,
    has one float32 scale per page and head.  A page's scale grows with its tokens, and its earlier codes are then
    rounded again; writing a page's first token begins its scale anew."""
    index, cache, heads, dim = _cache(k_cache, v_cache, k_scale, v_scale)
    if k.requires_grad or v.requires_grad:
        _no_gradient()
    tokens = k.shape[0]
    dtype = _DTYPES.get(k.dtype)
    if dtype is None or v.dtype is not k.dtype:
        raise TypeError(f"k and v must both be float32, float16 or bfloat16 (got {k.dtype}, {v.dtype})")
    size, ks, vs = (tokens, heads, dim), k.stride(), v.stride()
    if k.shape != size or v.shape != size or ks[2] != 1 or vs[2] != 1 or k.get_device() != index or v.get_device() != index:
        raise ValueError(f"k and v must be {size} on cuda:{index}, the last dimension contiguous (got {tuple(k.shape)}, "
                         f"{tuple(v.shape)})")
    _call(_library().ptowsp_cuda_kv8_append, index, cache, _pack_append(
        k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1], _vector(slots, "slots", torch.int64, tokens, index),
        tokens, dtype, 0, _vector(status, "status", torch.int32, 1, index)))


def attend_kv8(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_len, *, q_start=None, max_q: int | None = None, scale=None,
               window: int = 0, out=None, return_lse: bool = False, status=None):
    """Causal attention of each request's newest tokens over its cached ones.

    ``q`` [tokens, heads, head_dim] in float16 or bfloat16, one row per request, or rows ``q_start[r]`` ..
    ``q_start[r + 1] - 1`` (int32 [requests + 1]) of request r, at most ``max_q`` (unless given: all of them, which a
    batch of short requests pays for with the launches for long ones).  ``kv_len`` int32 [requests] counts
    the cached tokens, the new ones included, whose pages stand in ``page_table`` int32 [requests, max_pages].
    ``scale`` of the scores: 1 / sqrt(head_dim) unless given; ``window`` > 0: a row sees its own token and the
    window - 1 before it.  Returns out like q, and with ``return_lse`` also float32 [tokens, heads].  Rows that see no
    key, that no request has, or whose request has more than ``max_q`` (also reported) are zeros with an lse of -inf."""
    index, cache, _, dim = _cache(k_cache, v_cache, k_scale, v_scale)
    if q.requires_grad:
        _no_gradient()
    dtype = _DTYPES.get(q.dtype)
    if not dtype:
        raise TypeError(f"q must be float16 or bfloat16 (got {q.dtype})")
    shape, qs = q.shape, q.stride()
    if len(shape) != 3 or shape[2] != dim or qs[2] != 1 or q.get_device() != index:
        raise ValueError(f"q must be [tokens, heads, {dim}] on cuda:{index}, the last dimension contiguous (got {tuple(shape)})")
    tokens, heads, _ = shape
    if out is None:
        out, os = q.new_empty(shape), (heads * dim, dim, 1)
    else:
        os = out.stride()
        if out.shape != shape or out.dtype is not q.dtype or out.get_device() != index or os[2] != 1:
            raise ValueError("out must be like q")
    if max_q is None:
        max_q = 1 if q_start is None else tokens
    i32 = torch.int32
    requests = kv_len.shape[0]
    table, stride, max_pages = _table(page_table, requests, index)
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    # all but the workspace, its size and the status
    head = (q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, qs[0], qs[1], os[0], os[1], table, stride,
            _vector(kv_len, "kv_len", i32, requests, index), _vector(q_start, "q_start", i32, requests + 1, index), tokens,
            max_pages, requests, heads, max_q, window, dtype, dim ** -0.5 if scale is None else scale, 0)
    lib = _library()
    a = _pack_attention(*head, 0, 0, 0)
    if index == torch._C._cuda_getDevice():
        nbytes = lib.ptowsp_cuda_kv8_attention_workspace(cache, a)
    else:
        with torch.cuda.device(index):
            nbytes = lib.ptowsp_cuda_kv8_attention_workspace(cache, a)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    _call(lib.ptowsp_cuda_kv8_attention, index, cache,
          _pack_attention(*head, workspace.data_ptr(), nbytes, _vector(status, "status", i32, 1, index)))
    return (out, lse) if return_lse else out


def sample_tokens(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token per row of ``logits`` [rows, vocab] (float32, float16 or bfloat16) from the uniform random numbers
    ``u`` float32 [rows] in [0, 1).

    Per-row settings, each may be None: ``temperature`` float32 (0: the largest logit), ``top_k`` int32 (0: all),
    ``top_p`` float32 (1: all), ``min_p`` float32 (0: all), applied in the order temperature, top-k, min-p, top-p.
    Returns the tokens, int32 [rows] (-1 where every logit is -inf or NaN), and the logarithm of each one's
    probability among what the settings left, float32 [rows]."""
    index = _cuda_index(logits, "logits")
    if logits.requires_grad:
        _no_gradient()
    dtype = _DTYPES.get(logits.dtype)
    if dtype is None:
        raise TypeError(f"logits must be float32, float16 or bfloat16 (got {logits.dtype})")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [rows, vocab], its rows contiguous")
    rows, vocab = logits.shape
    f32 = torch.float32
    at_u = _vector(u, "u", f32, rows, index)
    logprob = torch.empty_like(u)
    token = torch.empty_like(u, dtype=torch.int32)
    _call(_library().ptowsp_cuda_sample_tokens, index, _pack_sample(
        logits.data_ptr(), logits.stride(0), rows, vocab, dtype, 0, at_u,
        _vector(temperature, "temperature", f32, rows, index), _vector(top_k, "top_k", torch.int32, rows, index),
        _vector(top_p, "top_p", f32, rows, index), _vector(min_p, "min_p", f32, rows, index), token.data_ptr(),
        logprob.data_ptr()))
    return token, logprob
