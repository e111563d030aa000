"""Queries and keys on their way into attention: per-head RMS norm and position rotation in one pass.

`qk_norm_rope` is what `llama.RandomLlama` runs on every layer's projected queries and keys, at prefill
(many tokens per request) and at decode (one).  `kv4.rope_append` is the same pass with the keys and
values written into a 4-bit cache.  Forward only; runs on the current CUDA stream of q's device.
"""
from __future__ import annotations

import torch

from . import _lib
from .geometry import D

_CODE = {torch.bfloat16: _lib.OA_BF16, torch.float32: _lib.OA_F32}

# None on a torch without CUDA, where every call is refused (its tensors are not on a GPU) before it gets here
_current_device = getattr(torch._C, "_cuda_getDevice", None)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _bad_rows(name, t, dtype, dev):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 4:
        raise RuntimeError(f"{name} must be (B, heads, T, 128), got {tuple(t.shape)}")
    if t.get_device() != dev:
        raise RuntimeError(f"{name} must be a tensor on cuda:{dev}, got {t.device}")
    _no_grad(name, t)


def _no_grad(name, t):
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient: this operator has no backward pass (use torch.no_grad())")


def _rows(name, t, dtype, dev):
    """The block's fields of (B, heads, T, 128) rows on GPU `dev`; sizes, strides and alignment are checked by the
    entry.  Every call of a decode step comes through here: one expression, and the message is made apart."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype is not dtype or t.dim() != 4 or \
            t.get_device() != dev or (t.requires_grad and torch.is_grad_enabled()):
        _bad_rows(name, t, dtype, dev)
    return t.data_ptr(), *t.shape, *t.stride()


def _device_of(name, t):
    """The GPU of a call's leading tensor."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _same_device(dev, **tensors):
    for name, t in tensors.items():
        if t is not None and (not isinstance(t, torch.Tensor) or t.get_device() != dev):
            where = t.device if isinstance(t, torch.Tensor) else type(t).__name__
            raise RuntimeError(f"{name} must be a tensor on cuda:{dev}, got {where}")


def _index(name, t, dev):
    """The block's fields of one whole number for each request, or one for all."""
    if t is None:
        return 0, 0, 0, 0
    if not isinstance(t, torch.Tensor) or t.get_device() != dev or t.dim() != 1 or \
            (t.dtype is not torch.int32 and t.dtype is not torch.int64):
        got = f"{tuple(t.shape)} {t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise RuntimeError(f"{name} must be (B,) or (1,) int32 or int64 on cuda:{dev}, got {got}")
    return t.data_ptr(), t.shape[0], t.stride(0), t.dtype is torch.int64


def _bad_table(cos, sin, dev):
    for name, t in (("cos", cos), ("sin", sin)):
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.float32 or t.get_device() != dev or t.dim() != 2 or \
                not t.is_contiguous() or (t is not cos and t.shape != cos.shape):
            raise RuntimeError(f"{name} must be a contiguous fp32 (positions, rotated dims) table on cuda:{dev}, the "
                               "same shape for both")
        _no_grad(name, t)


def _table(cos, sin, dev):
    try:
        shape = cos.shape
        if sin.shape == shape and cos.dtype is sin.dtype is torch.float32 and cos.get_device() == sin.get_device() == dev and \
                cos.is_contiguous() and sin.is_contiguous() and not (cos.requires_grad or sin.requires_grad):
            rows, width = shape
            return cos.data_ptr(), sin.data_ptr(), rows, width
    except (AttributeError, ValueError):
        pass
    _bad_table(cos, sin, dev)
    return cos.data_ptr(), sin.data_ptr(), *cos.shape


def _weights(q_weight, k_weight, dtype, dev):
    """(q pointer, k pointer, dtype code) of the norm weights: both in the rows' type or both fp32."""
    if q_weight is None and k_weight is None:
        return 0, 0, _lib.OA_F32
    given = [w for w in (q_weight, k_weight) if w is not None]
    for w in given:
        if not isinstance(w, torch.Tensor) or w.get_device() != dev or w.shape != (D,) or not w.is_contiguous() or \
                w.dtype not in (dtype, torch.float32) or w.dtype != given[0].dtype:
            raise RuntimeError(f"norm weights must be contiguous ({D},) tensors on cuda:{dev}, both {dtype} or both fp32")
        _no_grad("a norm weight", w)
    return _lib.ptr(q_weight), _lib.ptr(k_weight), _CODE[given[0].dtype]


def _like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _own_rows(t, sizes):
    """_rows of a contiguous tensor that the call itself allocated; sizes: (B, heads, T, 128)."""
    _, H, T, _ = sizes
    return t.data_ptr(), *sizes, H * T * D, T * D, D, 1


_entries: dict = {}


def _call(dev, name, *fields):
    """An entry with its argument block, on the current stream of GPU `dev` (a launch needs its stream's device to be
    current)."""
    entry = _entries.get(name)
    if entry is None:
        entry = _entries[name] = _lib.block_entry(name)
    if dev == _current_device():
        status = entry[1](entry[0](*fields), _current_stream(dev))
    else:
        with torch.cuda.device(dev):
            status = entry[1](entry[0](*fields), _current_stream(dev))
    if status:
        _lib.fail(name, status)


def qk_norm_rope(q, k, cos, sin, start, *, offset=0, lens=None, q_weight=None, k_weight=None, eps=1e-5, q_out=None,
                 k_out=None):
    """q (B, HQ, T, 128), k (B, HKV, T, 128) -> the normalised, rotated (q, k).

    Row i of request b stands at position p = start[b] + offset + i:
        y = x * rsqrt(mean(x^2) + eps) * weight     (fp32; only where q_weight / k_weight (128,) is given)
        out[d] = y[d] * cos[p, d] + rot(y)[d] * sin[p, d]  for d < R, y[d] for the other dims,
    rot(y) = [-y[R/2:R], y[:R/2]], rounded once to the rows' type.  q and k are bf16 or fp32 with any strides
    (a contiguous last dim, rows on 16-byte boundaries); cos, sin (P, R) fp32, R a multiple of 16 up to 128;
    start and lens are device arrays, (B,) or (1,), int32 or int64.

    lens[b] (default T) rows of request b are real.  Rows behind them, and rows whose position is outside
    the table, are padding: they are zero in outputs that this call allocates and left as they were in
    q_out / k_out.  q_out may be q and k_out may be k (in place); otherwise outputs must not overlap inputs."""
    dev = _device_of("q", q)
    dt = torch.float32 if q.dtype is torch.float32 else torch.bfloat16
    fq, fk = _rows("q", q, dt, dev), _rows("k", k, dt, dev)
    zq, zk = q_out is None, k_out is None
    if zq:
        q_out = _like(q)
        fqo = _own_rows(q_out, fq[1:5])
    else:
        fqo = _rows("q_out", q_out, dt, dev)
    if zk:
        k_out = _like(k)
        fko = _own_rows(k_out, fk[1:5])
    else:
        fko = _rows("k_out", k_out, dt, dev)
    qp, kp, wd = _weights(q_weight, k_weight, dt, dev)
    _call(dev, "oa_qk_norm_rope", *fq, *fk, *fqo, *fko, *_table(cos, sin, dev), *_index("start", start, dev), *_index("lens", lens, dev), qp, kp, offset, _CODE[dt], wd,
          zq, zk, eps)
    return q_out, k_out
