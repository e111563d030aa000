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


def _rows(name, t, dtype, shape=None):
    """(B, heads, T, 128) rows whose last dim is contiguous, on CUDA; any other strides."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 4 or t.shape[3] != D or t.stride(3) != 1 or (shape is not None and t.shape != shape):
        want = "(B, heads, T, 128)" if shape is None else tuple(shape)
        raise RuntimeError(f"{name} must be {want} with a contiguous last dim, got {tuple(t.shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient: this operator has no backward pass (use torch.no_grad())")


def _same_device(dev, **tensors):
    for name, t in tensors.items():
        if t is not None and (not isinstance(t, torch.Tensor) or t.device != dev):
            where = t.device if isinstance(t, torch.Tensor) else type(t).__name__
            raise RuntimeError(f"{name} must be a tensor on {dev}, got {where}")


def _strides(t):
    """Strides of the first three dims; a dim of one element has none."""
    if t is None:
        return 0, 0, 0
    return tuple(0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3]))


def _out(name, t, dtype, shape):
    """An output's rows must not overlap each other (an expanded tensor would be written by several rows)."""
    _rows(name, t, dtype, shape)
    if any(s == 0 and n > 1 for n, s in zip(t.shape, t.stride())):
        raise RuntimeError(f"{name} must not be an expanded tensor")


def _per_request(name, t, B, dev):
    """(pointer, stride, is_int64) of one whole number for each request, or one for all."""
    if t is None:
        return 0, 0, 0
    if not isinstance(t, torch.Tensor) or t.device != dev or t.dtype not in (torch.int32, torch.int64) or t.dim() != 1 \
            or t.shape[0] not in (1, B):
        got = f"{tuple(t.shape)} {t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise RuntimeError(f"{name} must be ({B},) or (1,) int32 or int64 on {dev}, got {got}")
    return t.data_ptr(), 0 if t.shape[0] == 1 else t.stride(0), 1 if t.dtype == torch.int64 else 0


def _table(cos, sin, dev):
    for name, t in (("cos", cos), ("sin", sin)):
        if not isinstance(t, torch.Tensor) or t.device != dev or t.dtype != torch.float32 or t.dim() != 2 or \
                not t.is_contiguous() or t.shape != cos.shape:
            raise RuntimeError(f"{name} must be a contiguous fp32 (positions, rotated dims) table on {dev}, the same "
                               "shape for both")
    return cos.data_ptr(), sin.data_ptr(), cos.shape[0], cos.shape[1]


def _weights(q_weight, k_weight, dtype, dev):
    """(q pointer, k pointer, dtype code) of the norm weights: both in the rows' type or both fp32."""
    given = [w for w in (q_weight, k_weight) if w is not None]
    for w in given:
        if not isinstance(w, torch.Tensor) or w.device != dev or w.shape != (D,) or not w.is_contiguous() or \
                w.dtype not in (dtype, torch.float32) or w.dtype != given[0].dtype:
            raise RuntimeError(f"norm weights must be contiguous ({D},) tensors on {dev}, both {dtype} or both fp32")
    return _lib.ptr(q_weight), _lib.ptr(k_weight), _CODE[given[0].dtype] if given else _lib.OA_F32


def _call(dev, name, *args):
    """_lib.call on the current stream of `dev` (a launch needs its stream's device to be current)."""
    if dev.index == torch.cuda.current_device():
        _lib.call(name, *args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, torch.cuda.current_stream(dev).cuda_stream)


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
    _rows("q", q, q.dtype if getattr(q, "dtype", None) in _CODE else torch.bfloat16)
    dev, (B, HQ, T, _) = q.device, q.shape
    _rows("k", k, q.dtype, (B, k.shape[1], T, D) if isinstance(k, torch.Tensor) and k.dim() == 4 else None)
    _same_device(dev, k=k, q_out=q_out, k_out=k_out)
    tab = _table(cos, sin, dev)
    st, ln = _per_request("start", start, B, dev), _per_request("lens", lens, B, dev)
    wts = _weights(q_weight, k_weight, q.dtype, dev)
    zq, zk = q_out is None, k_out is None
    if zq:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _out("q_out", q_out, q.dtype, q.shape)
    if zk:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    else:
        _out("k_out", k_out, k.dtype, k.shape)
    p = _lib.ptr
    _call(dev, "oa_qk_norm_rope", p(q), *_strides(q), p(k), *_strides(k), p(q_out), *_strides(q_out), p(k_out),
          *_strides(k_out), _CODE[q.dtype], B, T, HQ, k.shape[1], *tab, *st, int(offset), *ln, *wts, float(eps),
          int(zq), int(zk))
    return q_out, k_out
