"""The operators beside the causal softmax on torch tensors (include/causal_attention.h).

Biased causal softmax with its gradient, and attention with a sliding window
and sinks (prompts, single tokens over a cache, training). Plumbing like the
rest of the binding: arguments are checked, outputs and workspaces are torch
allocations, and the work goes to the C entry points on `stream` (a torch
stream or a cudaStream_t; the current stream by default). With a `stream` of
its own, allocations belong to that stream; ordering the inputs before it, and
the outputs' use after it, is the caller's, as with any torch stream.

A query at position p sees the keys k <= p with p - k < window (window 0: all
of them) or k < sinks.

No call records an autograd graph: what comes back does not require a gradient,
whatever the inputs do. Training calls the *_backward function itself, or from the
backward of a torch.autograd.Function.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import struct

import torch

from . import check, lib

_I32_MAX = 2**31 - 1
_MAX_BUCKETS = 128  # CS_MAX_BUCKETS


class _BiasArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("type", "batch", "heads", "rows", "cols", "pitch", "row_offset",
                                              "window", "sinks", "buckets")] + \
        [("bucket_starts", ctypes.c_void_p), ("scale", ctypes.c_float)]


class _Tensor(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("batch_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64)]


class _AttentionArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("type", "batch", "heads", "kv_heads", "head_dim", "q_len", "kv_len",
                                              "window", "sinks")] + \
        [("scale", ctypes.c_float), ("q_lens", ctypes.c_void_p), ("kv_lens", ctypes.c_void_p),
         ("q", _Tensor), ("k", _Tensor), ("v", _Tensor), ("o", _Tensor), ("lse", ctypes.c_void_p)]


class _AttentionGrads(ctypes.Structure):
    _fields_ = [(n, _Tensor) for n in ("d_o", "dq", "dk", "dv")]


# The same layouts for struct: filling a ctypes structure field by field would
# take most of a small call's time.
_PACK_BIAS = struct.Struct("@10iPf4x").pack
_PACK_ATTENTION = struct.Struct("@9if2P" + "P3q" * 4 + "P").pack
_PACK_GRADS = struct.Struct("@" + "P3q" * 4).pack

_TYPES = {torch.float16: 0, torch.bfloat16: 1}

_library = None


def _lib():
    """The library, without the loader's lock once it is there."""
    global _library
    if _library is None:
        _library = lib()
    return _library


class _On:
    """A launch stream other than the current one of the current device, made current
    (with its device) while a call allocates and launches."""

    def __init__(self, device, stream):
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
        if stream is None:  # the device's current stream
            self._ctx = torch.cuda.device(device)
        elif stream.device != device:
            raise ValueError(f"stream of {stream.device} for tensors of {device}")
        else:
            self._ctx = torch.cuda.stream(stream)

    def __enter__(self):
        self._ctx.__enter__()

    def __exit__(self, *exc):
        self._ctx.__exit__(*exc)


_HERE = contextlib.nullcontext()


def _on(device, stream):
    return _HERE if stream is None and device.index == torch.cuda.current_device() else _On(device, stream)


def _current(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _int(name: str, v) -> int:
    if not -_I32_MAX <= v <= _I32_MAX:
        raise ValueError(f"{name} {v} does not fit 32 bits")
    n = int(v)
    if n != v:
        raise ValueError(f"{name} {v} is not a whole number")
    return n


def _same(name: str, t, dtype, device) -> None:
    if t.dtype != dtype or t.device != device:
        raise TypeError(f"{name} must be {dtype} on {device}, not {t.dtype} on {t.device}")


def _sixteen_bit(name: str, t) -> int:
    kind = _TYPES.get(t.dtype)
    if kind is None or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA float16 or bfloat16 tensor, not {t.dtype} on {t.device}")
    return kind


# ---------------------------------------------------------------- biased softmax

def bias_buckets(buckets: int, max_distance: int) -> tuple[int, ...]:
    """First distance of each bucket: half of them hold one distance each, the
    rest grow by an even ratio up to max_distance; the last holds all beyond."""
    n = _int("buckets", buckets)
    starts = (ctypes.c_int32 * _MAX_BUCKETS)()
    check(lib().cs_bias_buckets(n, _int("max_distance", max_distance), starts), "cs_bias_buckets")
    return tuple(starts[:n])


@functools.lru_cache(maxsize=64)
def _starts_array(starts: tuple):
    return (ctypes.c_int32 * max(1, len(starts)))(*(_int("bucket start", s) for s in starts))


def _bias_args(x, starts, cols, scale, row_offset, window, sinks):
    """The packed cs_bias_args, and (batch, heads, buckets). The starts' array outlives the call in the cache
    of its values, or in the frame that holds the result's last item."""
    kind = _sixteen_bit("the matrices", x)
    shape = x.shape
    if len(shape) not in (3, 4):
        raise ValueError("matrices are [batch,] heads, rows, pitch")
    if not x.is_contiguous():
        raise ValueError("matrices must be contiguous")
    batch = shape[0] if len(shape) == 4 else 1
    heads, rows, pitch = shape[-3:]
    starts = tuple(starts)
    array = _starts_array(starts)
    args = _PACK_BIAS(kind, _int("batch", batch), _int("heads", heads), _int("rows", rows), _int("cols", cols),
                      _int("pitch", pitch), _int("row_offset", row_offset), _int("window", window),
                      _int("sinks", sinks), len(starts), ctypes.addressof(array), scale)
    return args, heads, len(starts), array


def _like(name, out, x):
    if out is None:
        return torch.empty_like(x)
    _same(name, out, x.dtype, x.device)
    if out.shape != x.shape or not out.is_contiguous():
        raise ValueError(f"{name} must be contiguous, of shape {tuple(x.shape)}")
    return out


def bias_softmax(x, table, bucket_starts, *, cols: int, scale: float, row_offset: int = 0, window: int = 0,
                 sinks: int = 0, out=None, stream=None):
    """softmax(scale x + table[head, bucket(position - key)]) over each row's visible keys.

    x: float16 or bfloat16 [batch,] heads, rows, pitch (pitch % 8 == 0); row i is
    position row_offset + i. table: float32 heads, buckets. bucket_starts: the
    buckets' first distances (bias_buckets, or any ascending ones from 0).
    Every other column of the result, padding included, is +0.0. Autograd stops
    here; bias_softmax_backward has the gradients."""
    args, heads, buckets, _keep = _bias_args(x, bucket_starts, cols, scale, row_offset, window, sinks)
    device = x.device
    _same("table", table, torch.float32, device)
    if table.shape != (heads, buckets) or not table.is_contiguous():
        raise ValueError(f"table must be contiguous, [{heads}, {buckets}]")
    with _on(device, stream):
        out = _like("out", out, x)
        check(_lib().cs_bias_softmax(args, x.data_ptr(), table.data_ptr(), out.data_ptr(), _current(device)),
              "cs_bias_softmax")
    return out


def bias_softmax_backward(p, dp, bucket_starts, *, cols: int, scale: float, row_offset: int = 0, window: int = 0,
                          sinks: int = 0, out=None, stream=None):
    """Gradients of bias_softmax from its result p and dp, the gradient of p: (ds, dtable).

    ds: of the scores x, in their type (masked columns +0.0); dtable: float32
    heads, buckets, summed over the batch and the rows."""
    args, heads, buckets, _keep = _bias_args(p, bucket_starts, cols, scale, row_offset, window, sinks)
    device = p.device
    _same("dp", dp, p.dtype, device)
    if dp.shape != p.shape or not dp.is_contiguous():
        raise ValueError(f"dp must be contiguous, of shape {tuple(p.shape)}")
    L = _lib()
    with _on(device, stream):
        ds = _like("out", out, p)
        dtable = torch.empty(heads, buckets, dtype=torch.float32, device=device)
        need = L.cs_bias_softmax_backward_workspace(args)
        check(min(need, 0), "cs_bias_softmax_backward_workspace")
        work = torch.empty(need, dtype=torch.uint8, device=device)
        check(L.cs_bias_softmax_backward(args, p.data_ptr(), dp.data_ptr(), ds.data_ptr(), dtable.data_ptr(),
                                         work.data_ptr(), need, _current(device)), "cs_bias_softmax_backward")
    return ds, dtable


# ---------------------------------------------------------------- attention

def _tensor(name: str, t, shape, dtype, device) -> tuple:
    """data, batch_stride, token_stride, head_stride."""
    if t.dtype is not dtype or t.get_device() != device.index:
        raise TypeError(f"{name} must be {dtype} on {device}, not {t.dtype} on {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    b, n, h, d = t.stride()
    if d != 1 and shape[3] > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return t.data_ptr(), b, n, h


def _fresh(t):
    """A contiguous tensor like t. (empty_like takes 1.3 us, empty with a shape and a device 3.3.)"""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _lens(name: str, t, batch: int, device) -> int:
    if t is None:
        return 0
    _same(name, t, torch.int32, device)
    if t.shape != (batch,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous, [{batch}]")
    return t.data_ptr()


def _attention_head(q, k, v, scale, window, sinks, q_lens, kv_lens) -> tuple:
    """The fields of cs_attention_args up to v."""
    kind = _sixteen_bit("q", q)
    shape, dtype, device = q.shape, q.dtype, q.device
    if len(shape) != 4 or k.dim() != 4:
        raise ValueError("q, k and v are batch, tokens, heads, head_dim")
    batch, q_len, heads, dim = shape
    _, kv_len, kv_heads, _ = k.shape
    kv_shape = (batch, kv_len, kv_heads, dim)
    if max(batch, q_len, heads, dim, kv_len, kv_heads) > _I32_MAX:
        raise ValueError(f"sizes of q {list(shape)} and k {list(k.shape)} do not fit 32 bits")
    return (kind, batch, heads, kv_heads, dim, q_len, kv_len, _int("window", window), _int("sinks", sinks),
            max(1, dim) ** -0.5 if scale is None else scale,
            _lens("q_lens", q_lens, batch, device), _lens("kv_lens", kv_lens, batch, device),
            *_tensor("q", q, shape, dtype, device), *_tensor("k", k, kv_shape, dtype, device),
            *_tensor("v", v, kv_shape, dtype, device))


def attention(q, k, v, *, scale: float | None = None, window: int = 0, sinks: int = 0, q_lens=None, kv_lens=None,
              out=None, return_lse: bool = False, stream=None):
    """softmax(scale q k^T) v over each query's visible keys.

    q: float16 or bfloat16 batch, q_len, heads, head_dim; k, v: batch, kv_len,
    kv_heads, head_dim (heads a multiple of kv_heads, head_dim a multiple of 8 up
    to 128), any strides in multiples of 8 with the last dimension contiguous.
    scale: 1 / sqrt(head_dim) by default. q_lens, kv_lens: int32 [batch] on the
    device, the sequences' lengths (the tensors' by default); a sequence's queries
    are its last tokens, so q_len 1 with kv_lens reads a cache. Rows behind a
    sequence's queries come back zero. Returns out, or (out, lse) with the float32
    log-sum-exp [batch, heads, q_len] that attention_backward takes. Autograd stops
    here; attention_backward has the gradients."""
    head = _attention_head(q, k, v, scale, window, sinks, q_lens, kv_lens)
    shape, dtype, device = q.shape, q.dtype, q.device
    L = _lib()
    with _on(device, stream):
        if out is None:
            out = _fresh(q)
        lse = torch.empty((shape[0], shape[2], shape[1]), dtype=torch.float32, device=device) if return_lse else None
        args = _PACK_ATTENTION(*head, *_tensor("out", out, shape, dtype, device), lse.data_ptr() if return_lse else 0)
        need = L.cs_attention_workspace(args)
        check(min(need, 0), "cs_attention_workspace")
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        check(L.cs_attention(args, work.data_ptr() if need else None, need, _current(device)), "cs_attention")
    return (out, lse) if return_lse else out


def attention_backward(dout, q, k, v, out, lse, *, scale: float | None = None, window: int = 0, sinks: int = 0,
                       q_lens=None, kv_lens=None, stream=None):
    """(dq, dk, dv) from dout, the gradient of attention's out, with the out and lse of the same arguments."""
    head = _attention_head(q, k, v, scale, window, sinks, q_lens, kv_lens)
    shape, dtype, device = q.shape, q.dtype, q.device
    _same("lse", lse, torch.float32, device)
    if lse.shape != (shape[0], shape[2], shape[1]) or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous, {[shape[0], shape[2], shape[1]]}")
    args = _PACK_ATTENTION(*head, *_tensor("out", out, shape, dtype, device), lse.data_ptr())
    d_o = _tensor("dout", dout, shape, dtype, device)
    L = _lib()
    with _on(device, stream):
        dq, dk, dv = _fresh(q), _fresh(k), _fresh(v)
        grads = _PACK_GRADS(*d_o, dq.data_ptr(), *dq.stride()[:3], dk.data_ptr(), *dk.stride()[:3],
                            dv.data_ptr(), *dv.stride()[:3])
        need = L.cs_attention_backward_workspace(args)
        check(min(need, 0), "cs_attention_backward_workspace")
        work = torch.empty(need, dtype=torch.uint8, device=device)
        check(L.cs_attention_backward(args, grads, work.data_ptr(), need, _current(device)), "cs_attention_backward")
    return dq, dk, dv


def attention_status(stream=None, device=None) -> tuple[int, int]:
    """(error code, bits) of the attention kernels' status word on a device, which it clears; waits for the stream."""
    index = None if device is None else torch.device(device).index
    device = torch.device("cuda", torch.cuda.current_device() if index is None else index)
    bits = ctypes.c_uint32()
    with _on(device, stream):
        rc = lib().cs_attention_status(ctypes.byref(bits), _current(device))
    return rc, bits.value
