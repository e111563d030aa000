"""A K/V cache held in 4 bits, and attention over it.

    cache = kv4.new_cache(B, Lmax, dev)                       # (B, 8, Lmax, 144) uint8: 3.6x smaller than bf16 K and V
    kv4.append(cache, k, v, start)                            # prompt rows (keys already rotated)
    q = kv4.rope_append(cache, q, k, v, cos, sin, start)      # or: norm + rotate q and k, write k and v, one launch
    out = kv4.decode_attention(q, cache, n)                   # dense, over every request's n positions
    out = kv4.flash_attention(q, cache, sel, exp, kbar, vbar, log_n)  # flash.ours_flash's lists over this cache
    k, v = kv4.unpack(cache, start, T)                        # rows back as bf16 (to re-prefill, to compare)

One record is one token of one KV head in 144 bytes: 64 bytes of K codes, 64 of V codes, and (scale, offset) in
bf16 for dims 0..63 and 64..127 of K, then of V.  Byte j holds the code of dim j in its low nibble and of dim
j + 64 in its high one; a value is scale * code + offset.  The offset is the group's minimum, the scale
bf16((max - min) / 15), the code min(rint((x - offset) / scale), 15), so a value is off by at most about half a
scale.  A group that holds an infinity or a NaN reads back as NaN.

Positions are device arrays (int32 or int64, one for each request or one for all), so every call can be captured
in a CUDA graph and replayed as they advance.  Forward only; everything runs on the current CUDA stream.
"""
from __future__ import annotations

import torch

from . import _lib
from .geometry import D, HKV
from .rotary import _call, _CODE, _out, _per_request, _rows, _same_device, _strides, _table, _weights

REC = 144


def new_cache(B, Lmax, dev, hkv=HKV):
    """(B, hkv, Lmax, 144) uint8 records; all zero, which reads as zeros."""
    return torch.zeros(B, hkv, Lmax, REC, dtype=torch.uint8, device=dev)


def _cache(cache, ndim=4, write=False):
    if not isinstance(cache, torch.Tensor) or not cache.is_cuda:
        raise RuntimeError("cache must be a CUDA tensor")
    if cache.dtype != torch.uint8 or cache.dim() != ndim or cache.shape[-1] != REC or cache.stride(-1) != 1 or \
            (cache.shape[-2] > 1 and cache.stride(-2) != REC):
        raise RuntimeError(f"cache must be {'(B, hkv, Lmax, 144)' if ndim == 4 else '(B * hkv, Lmax, 144)'} uint8 with "
                           f"contiguous records, got {tuple(cache.shape)} {cache.dtype} strides {cache.stride()}")
    if write and any(s == 0 and n > 1 for n, s in zip(cache.shape, cache.stride())):
        raise RuntimeError("cache must not be an expanded tensor: its requests would share records")


def _hstrides(cache):
    return tuple(0 if n == 1 else s for n, s in zip(cache.shape[:-2], cache.stride()[:-2]))


def _append(cache, q, k, v, cos, sin, start, offset, lens, q_weight, k_weight, eps, q_out):
    _cache(cache, write=True)
    dev, (B, hkv, Lmax, _) = cache.device, cache.shape
    _rows("k", k, torch.bfloat16, (B, hkv, k.shape[2], D) if isinstance(k, torch.Tensor) and k.dim() == 4 else None)
    T = k.shape[2]
    _rows("v", v, torch.bfloat16, k.shape)
    _same_device(dev, k=k, v=v, q=q, q_out=q_out)
    st, ln = _per_request("start", start, B, dev), _per_request("lens", lens, B, dev)
    tab, wts, HQ, zq = (0, 0, 0, 0), (0, 0, _lib.OA_F32), 0, False
    if start is None:
        raise RuntimeError("start must be given: the position of each request's first row")
    if q is not None:
        _rows("q", q, torch.bfloat16, (B, q.shape[1], T, D) if q.dim() == 4 else None)
        HQ = q.shape[1]
        tab, wts, zq = _table(cos, sin, dev), _weights(q_weight, k_weight, torch.bfloat16, dev), q_out is None
        if zq:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            _out("q_out", q_out, q.dtype, q.shape)
    p = _lib.ptr
    _call(dev, "oa_kv4_append", p(q), *_strides(q), p(k), *_strides(k), p(v), *_strides(v), p(q_out), *_strides(q_out),
          p(cache), *_hstrides(cache), Lmax, B, T, HQ, hkv, *tab, *st, int(offset), *ln, *wts, float(eps), int(zq))
    return q_out


def append(cache, k, v, start, *, offset=0, lens=None):
    """Writes k, v (B, hkv, T, 128) bf16 into the cache (B, hkv, Lmax, 144): row i of request b at position
    start[b] + offset + i.  Rows i >= lens[b] (default T) and positions outside [0, Lmax) write nothing.
    Calls that write the same positions must be ordered (one stream, or events)."""
    _append(cache, None, k, v, None, None, start, offset, lens, None, None, 0.0, None)


def rope_append(cache, q, k, v, cos, sin, start, *, offset=0, lens=None, q_weight=None, k_weight=None, eps=1e-5,
                q_out=None):
    """rotary.qk_norm_rope and append in one launch: returns the normalised, rotated q (B, HQ, T, 128) bf16 and
    writes the normalised, rotated k (rounded to bf16) and v into the cache.  Arguments as in those two; rows
    whose position is outside the tables or behind lens are padding (no record; q as in qk_norm_rope), rows at
    positions past the cache rotate q and write no record."""
    if not isinstance(q, torch.Tensor):
        raise RuntimeError("q must be a CUDA tensor")
    return _append(cache, q, k, v, cos, sin, start, offset, lens, q_weight, k_weight, eps, q_out)


def unpack(cache, start, T, *, offset=0, lens=None, out_dtype=torch.bfloat16, k_out=None, v_out=None):
    """The values (k, v), each (B, hkv, T, 128) bf16 or fp32, of the records at positions start[b] + offset + i,
    i < T.  Rows i >= lens[b] and positions outside the cache are zero in outputs that this call allocates and
    left as they were in k_out / v_out."""
    _cache(cache)
    dev, (B, hkv, Lmax, _) = cache.device, cache.shape
    if start is None:
        raise RuntimeError("start must be given: the position of each request's first row")
    if T < 0 or out_dtype not in _CODE:
        raise RuntimeError(f"T must be >= 0 and out_dtype bf16 or fp32, got {T}, {out_dtype}")
    st, ln = _per_request("start", start, B, dev), _per_request("lens", lens, B, dev)
    zk, zv = k_out is None, v_out is None
    shape = torch.Size((B, hkv, T, D))
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is not None:
            _same_device(dev, **{name: t})
            out_dtype = t.dtype if t.dtype in _CODE else out_dtype
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is not None:
            _out(name, t, out_dtype, shape)
    k_out = torch.empty(shape, dtype=out_dtype, device=dev) if zk else k_out
    v_out = torch.empty(shape, dtype=out_dtype, device=dev) if zv else v_out
    p = _lib.ptr
    _call(dev, "oa_kv4_unpack", p(cache), *_hstrides(cache), Lmax, *st, int(offset), *ln, p(k_out), *_strides(k_out),
          p(v_out), *_strides(v_out), _CODE[out_dtype], B, T, hkv, int(zk), int(zv))
    return k_out, v_out


_ws_cache: dict = {}


def attention_workspace(B, HQ, T, cache_len, dev, hkv=HKV):
    """Scratch of decode_attention for these sizes (uint8, zero-filled; None where it needs none).  Calls that
    can overlap on the GPU must not share one."""
    need = _lib.load().oa_kv4_attention_workspace_bytes(B, HQ, hkv, T, cache_len)
    return torch.zeros(need, dtype=torch.uint8, device=dev) if need else None


def decode_attention(q, cache, n, *, offset=0, sm_scale=None, out_dtype=None, out=None, workspace=None):
    """q (B, HQ, T, 128) bf16 over the cache (B, hkv, Lmax, 144) -> (B, HQ, T, 128) in out_dtype (bf16, the
    default, or fp32).

    n (B,) or (1,) int32 or int64 on the device: request b's length is min(n[b] + offset, Lmax), its T query
    tokens the last T positions; token i sees positions <= length - T + i.  HQ is a multiple of hkv, query head h
    reads KV head h // (HQ // hkv).  A query token before the first position (a length below T, zero or
    negative) gives zeros.  Records at positions >= the length are never used.  sm_scale defaults to 128**-0.5.

    workspace: attention_workspace(...) of the same sizes.  By default one is kept for each device, stream and
    size; a call that is being captured allocates its own from the graph's pool (graphs may then be replayed
    side by side), so a decode loop that captures many layers passes one."""
    _rows("q", q, torch.bfloat16)
    _cache(cache)
    dev, (B, HQ, T, _) = q.device, q.shape
    hkv, Lmax = cache.shape[1], cache.shape[2]
    if cache.shape[0] != B or hkv < 1 or HQ < 1 or HQ % hkv:
        raise RuntimeError(f"q holds {B} requests of {HQ} heads, the cache {cache.shape[0]} of {hkv}: need the same "
                           "requests and a multiple of the KV heads")
    _same_device(dev, cache=cache, out=out, workspace=workspace)
    if n is None:
        raise RuntimeError("n must be given: the length of each request")
    ln = _per_request("n", n, B, dev)
    if workspace is not None and (workspace.dtype != torch.uint8 or not workspace.is_contiguous()):
        raise RuntimeError("workspace must be a contiguous uint8 tensor")
    if out is None:
        out = torch.empty(q.shape, dtype=out_dtype or q.dtype, device=dev)
    elif out_dtype is not None and out_dtype != out.dtype:
        raise RuntimeError(f"out is {out.dtype}, out_dtype {out_dtype}")
    if out.dtype not in _CODE:
        raise RuntimeError(f"the output must be bf16 or fp32, got {out.dtype}")
    _out("out", out, out.dtype, q.shape)
    need = _lib.load().oa_kv4_attention_workspace_bytes(B, HQ, hkv, T, Lmax)
    if workspace is None and need:
        if torch.cuda.is_current_stream_capturing():
            workspace = torch.zeros(need, dtype=torch.uint8, device=dev)
        else:
            key = (dev.index, torch.cuda.current_stream(dev).cuda_stream, B, HQ, hkv, T, Lmax)
            workspace = _ws_cache.get(key)
            if workspace is None:
                workspace = _ws_cache[key] = torch.zeros(need, dtype=torch.uint8, device=dev)
    p = _lib.ptr
    _call(dev, "oa_kv4_attention", p(q), *_strides(q), p(cache), *_hstrides(cache), Lmax, *ln, int(offset), p(out),
          *_strides(out), _CODE[out.dtype], B, HQ, hkv, T, float(D ** -0.5 if sm_scale is None else sm_scale),
          p(workspace), 0 if workspace is None else workspace.numel())
    return out


def flash_attention(q, cache, sel_idx, exp_idx, kbar, vbar, log_n, nb=None, *, sm_scale=None, out_dtype=None,
                    out=None):
    """flash.ours_flash / flash.decode_expand_attention over a 4-bit cache: q (BQ, 128) bf16, cache (BH, Lmax, 144)
    -> (BQ, 128).  Row r reads KV row r // (BQ // BH).

    One softmax over the tokens of sel_idx (BQ, n_sel) and exp_idx (BQ, n_exp) (int32; an index outside [0, Lmax)
    is padding) and nb cluster proxies with logits q . kbar * sm_scale + log_n (log_n = -inf skips one).
    kbar, vbar bf16 (BQ, NB, 128) (for each query row) or (BH, NB, 128) (for each KV row), log_n (BQ, NB) fp32;
    nb = 0 disables the proxies.  A row with nothing to attend gives zeros."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda or q.dtype != torch.bfloat16 or q.dim() != 2 or \
            q.shape[1] != D or q.stride(1) != 1:
        raise RuntimeError("q must be a (rows, 128) bf16 CUDA tensor with a contiguous last dim")
    if q.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("q requires a gradient: this operator has no backward pass (use torch.no_grad())")
    _cache(cache, ndim=3)
    dev, BQ = q.device, q.shape[0]
    BH, Lmax, _ = cache.shape
    if BH < 1 or BQ % BH:
        raise RuntimeError(f"q's {BQ} rows must be a multiple of the cache's {BH}")
    _same_device(dev, cache=cache, sel_idx=sel_idx, exp_idx=exp_idx, out=out)
    for name, t in (("sel_idx", sel_idx), ("exp_idx", exp_idx)):
        if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != BQ or not t.is_contiguous():
            raise RuntimeError(f"{name} must be a contiguous ({BQ}, n) int32 tensor, got {tuple(t.shape)} {t.dtype}")
    NB = (0 if kbar is None else kbar.shape[1]) if nb is None else int(nb)
    if NB < 0:
        raise RuntimeError(f"nb must not be negative, got {NB}")
    per_qhead, strides = 1, (0, 0)
    if NB > 0:
        _same_device(dev, kbar=kbar, vbar=vbar, log_n=log_n)
        for name, t in (("kbar", kbar), ("vbar", vbar)):
            if t.dtype != torch.bfloat16 or t.dim() != 3 or t.shape[0] not in (BQ, BH) or t.shape[1] < NB or \
                    t.shape[2] != D or t.stride(2) != 1 or t.shape != kbar.shape or t.stride() != kbar.stride():
                raise RuntimeError(f"{name} must be ({BQ} or {BH}, >= {NB}, 128) bf16 with a contiguous last dim, kbar and "
                                   f"vbar of one shape and strides; got {tuple(t.shape)} {t.dtype}")
        if log_n.dtype != torch.float32 or log_n.dim() != 2 or log_n.shape[0] != BQ or log_n.shape[1] < NB or \
                log_n.stride(1) != 1:
            raise RuntimeError(f"log_n must be ({BQ}, >= {NB}) fp32 with a contiguous last dim, got {tuple(log_n.shape)}")
        per_qhead = 1 if kbar.shape[0] == BQ else 0
        strides = tuple(0 if m == 1 else s for m, s in zip(kbar.shape[:2], kbar.stride()[:2]))
    if out is None:
        out = torch.empty(BQ, D, dtype=out_dtype or q.dtype, device=dev)
    if out.dtype not in _CODE or out.shape != (BQ, D) or out.stride(1) != 1 or (BQ > 1 and out.stride(0) < D) or \
            (out_dtype is not None and out_dtype != out.dtype):
        raise RuntimeError(f"out must be ({BQ}, 128) bf16 or fp32 rows, got {tuple(out.shape)} {out.dtype}")
    p = _lib.ptr
    _call(dev, "oa_kv4_flash", p(q), q.stride(0) if BQ > 1 else 0, p(cache), *_hstrides(cache), Lmax, p(sel_idx),
          sel_idx.shape[1], p(exp_idx), exp_idx.shape[1], p(kbar) if NB else 0, p(vbar) if NB else 0, *strides, per_qhead,
          p(log_n) if NB else 0, log_n.stride(0) if NB else 0, p(out), out.stride(0) if BQ > 1 else 0, _CODE[out.dtype],
          BQ, BH, NB, float(D ** -0.5 if sm_scale is None else sm_scale))
    return out
