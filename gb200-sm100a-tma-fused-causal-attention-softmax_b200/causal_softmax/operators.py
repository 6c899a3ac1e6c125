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
"""
from __future__ import annotations

import ctypes
import functools
import math

from . import check, lib

_I32_MAX = 2**31 - 1


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


@functools.lru_cache(maxsize=None)
def _types():
    import torch

    return {torch.float16: 0, torch.bfloat16: 1}


class _On:
    """The tensors' device and the launch stream, current while the call allocates and launches."""

    def __init__(self, device, stream):
        import torch

        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
        if stream is None:  # the device's current stream
            self._ctx = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)
        else:
            if stream.device != device:
                raise ValueError(f"stream of {stream.device} for tensors of {device}")
            self._ctx = torch.cuda.stream(stream)
        self._device = device

    def __enter__(self):
        import torch

        if self._ctx is not None:
            self._ctx.__enter__()
        return torch.cuda.current_stream(self._device).cuda_stream

    def __exit__(self, *exc):
        if self._ctx is not None:
            self._ctx.__exit__(*exc)


def _int(name: str, v) -> int:
    if not -_I32_MAX <= v <= _I32_MAX:
        raise ValueError(f"{name} {v} does not fit 32 bits")
    return int(v)


def _same(name: str, t, dtype, device) -> None:
    if t.dtype != dtype or t.device != device:
        raise TypeError(f"{name} must be {dtype} on {device}, not {t.dtype} on {t.device}")


def _sixteen_bit(name: str, t) -> int:
    kind = _types().get(t.dtype)
    if kind is None or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA float16 or bfloat16 tensor, not {t.dtype} on {t.device}")
    return kind


# ---------------------------------------------------------------- biased softmax

def bias_buckets(buckets: int, max_distance: int) -> tuple[int, ...]:
    """First distance of each bucket: half of them hold one distance each, the
    rest grow by an even ratio up to max_distance; the last holds all beyond."""
    starts = (ctypes.c_int32 * max(1, buckets))()
    check(lib().cs_bias_buckets(_int("buckets", buckets), _int("max_distance", max_distance), starts),
          "cs_bias_buckets")
    return tuple(starts)


@functools.lru_cache(maxsize=64)
def _starts_array(starts: tuple):
    return (ctypes.c_int32 * max(1, len(starts)))(*starts)


def _bias_args(x, starts, cols, scale, row_offset, window, sinks) -> _BiasArgs:
    kind = _sixteen_bit("the matrices", x)
    if x.dim() not in (3, 4):
        raise ValueError("matrices are [batch,] heads, rows, pitch")
    if not x.is_contiguous():
        raise ValueError("matrices must be contiguous")
    batch = x.shape[0] if x.dim() == 4 else 1
    starts = tuple(starts)
    array = _starts_array(starts)
    args = _BiasArgs(kind, batch, x.shape[-3], x.shape[-2], _int("cols", cols), x.shape[-1],
                     _int("row_offset", row_offset), _int("window", window), _int("sinks", sinks), len(starts),
                     ctypes.addressof(array), scale)
    args.keep = array  # the structure holds only its address
    return args


def _like(name, out, x):
    import torch

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
    Every other column of the result, padding included, is +0.0."""
    import torch

    args = _bias_args(x, bucket_starts, cols, scale, row_offset, window, sinks)
    _same("table", table, torch.float32, x.device)
    if table.shape != (args.heads, args.buckets) or not table.is_contiguous():
        raise ValueError(f"table must be contiguous, [{args.heads}, {args.buckets}]")
    with _On(x.device, stream) as s:
        out = _like("out", out, x)
        check(lib().cs_bias_softmax(ctypes.byref(args), x.data_ptr(), table.data_ptr(), out.data_ptr(), s),
              "cs_bias_softmax")
    return out


def bias_softmax_backward(p, dp, bucket_starts, *, cols: int, scale: float, row_offset: int = 0, window: int = 0,
                          sinks: int = 0, out=None, stream=None):
    """Gradients of bias_softmax from its result p and dp, the gradient of p: (ds, dtable).

    ds: of the scores x, in their type (masked columns +0.0); dtable: float32
    heads, buckets, summed over the batch and the rows."""
    import torch

    args = _bias_args(p, bucket_starts, cols, scale, row_offset, window, sinks)
    _same("dp", dp, p.dtype, p.device)
    if dp.shape != p.shape or not dp.is_contiguous():
        raise ValueError(f"dp must be contiguous, of shape {tuple(p.shape)}")
    L = lib()
    with _On(p.device, stream) as s:
        ds = _like("out", out, p)
        dtable = torch.empty(args.heads, args.buckets, dtype=torch.float32, device=p.device)
        need = L.cs_bias_softmax_backward_workspace(ctypes.byref(args))
        check(min(need, 0), "cs_bias_softmax_backward_workspace")
        work = torch.empty(need, dtype=torch.uint8, device=p.device)
        check(L.cs_bias_softmax_backward(ctypes.byref(args), p.data_ptr(), dp.data_ptr(), ds.data_ptr(),
                                         dtable.data_ptr(), work.data_ptr(), need, s), "cs_bias_softmax_backward")
    return ds, dtable


# ---------------------------------------------------------------- attention

def _tensor(name: str, t, shape, like) -> _Tensor:
    if t.dtype != like.dtype or t.device != like.device:
        raise TypeError(f"{name} must be {like.dtype} on {like.device}, not {t.dtype} on {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    b, n, h, d = t.stride()
    if d != 1 and shape[3] > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return _Tensor(t.data_ptr(), b, n, h)


def _lens(name: str, t, batch: int, device):
    import torch

    if t is None:
        return None
    _same(name, t, torch.int32, device)
    if t.shape != (batch,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous, [{batch}]")
    return t.data_ptr()


def _attention_args(q, k, v, scale, window, sinks, q_lens, kv_lens) -> _AttentionArgs:
    kind = _sixteen_bit("q", q)
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q, k and v are batch, tokens, heads, head_dim")
    batch, q_len, heads, dim = q.shape
    kv_len, kv_heads = k.shape[1], k.shape[2]
    kv_shape = (batch, kv_len, kv_heads, dim)
    return _AttentionArgs(kind, batch, heads, kv_heads, dim, q_len, kv_len, _int("window", window),
                          _int("sinks", sinks), 1.0 / math.sqrt(max(1, dim)) if scale is None else scale,
                          _lens("q_lens", q_lens, batch, q.device), _lens("kv_lens", kv_lens, batch, q.device),
                          _tensor("q", q, q.shape, q), _tensor("k", k, kv_shape, q), _tensor("v", v, kv_shape, q))


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
    log-sum-exp [batch, heads, q_len] that attention_backward takes."""
    import torch

    args = _attention_args(q, k, v, scale, window, sinks, q_lens, kv_lens)
    L = lib()
    with _On(q.device, stream) as s:
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        args.o = _tensor("out", out, q.shape, q)
        lse = None
        if return_lse:
            lse = torch.empty(args.batch, args.heads, args.q_len, dtype=torch.float32, device=q.device)
            args.lse = lse.data_ptr()
        ref = ctypes.byref(args)
        need = L.cs_attention_workspace(ref)
        check(min(need, 0), "cs_attention_workspace")
        work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        check(L.cs_attention(ref, work.data_ptr() if need else None, need, s), "cs_attention")
    return (out, lse) if return_lse else out


def attention_backward(dout, q, k, v, out, lse, *, scale: float | None = None, window: int = 0, sinks: int = 0,
                       q_lens=None, kv_lens=None, stream=None):
    """(dq, dk, dv) from dout, the gradient of attention's out, with the out and lse of the same arguments."""
    import torch

    args = _attention_args(q, k, v, scale, window, sinks, q_lens, kv_lens)
    args.o = _tensor("out", out, q.shape, q)
    _same("lse", lse, torch.float32, q.device)
    if lse.shape != (args.batch, args.heads, args.q_len) or not lse.is_contiguous():
        raise ValueError(f"lse must be contiguous, [{args.batch}, {args.heads}, {args.q_len}]")
    args.lse = lse.data_ptr()
    L = lib()
    with _On(q.device, stream) as s:
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        grads = _AttentionGrads(_tensor("dout", dout, q.shape, q), _tensor("dq", dq, q.shape, q),
                                _tensor("dk", dk, k.shape, q), _tensor("dv", dv, v.shape, q))
        ref = ctypes.byref(args)
        need = L.cs_attention_backward_workspace(ref)
        check(min(need, 0), "cs_attention_backward_workspace")
        work = torch.empty(need, dtype=torch.uint8, device=q.device)
        check(L.cs_attention_backward(ref, ctypes.byref(grads), work.data_ptr(), need, s), "cs_attention_backward")
    return dq, dk, dv


def attention_status(stream=None, device=None) -> tuple[int, int]:
    """(error code, bits) of the attention kernels' status word on a device, which it clears; waits for the stream."""
    import torch

    device = torch.device("cuda", torch.cuda.current_device() if device is None else torch.device(device).index or 0)
    bits = ctypes.c_uint32()
    with _On(device, stream) as s:
        rc = lib().cs_attention_status(ctypes.byref(bits), s)
    return rc, bits.value
