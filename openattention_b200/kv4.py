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

Attention multiplies the codes on the tensor cores.  There the product of a token's weight and its V scale is rounded
to fp16, 11 bits, in fp32 outputs too: a result is off by up to 2^-11 of the sum of weight * 15 * scale over its
tokens (5e-4 of it is typical for unit normal values), and fp32 outputs save the last rounding only.  Softmax maxima and
sums, offsets and proxies stay in fp32 (proxies' weights 16 bits).  The sum of weight * value is formed before it is
divided by the weights' sum, so values whose sum passes fp32 overflow.  Elements of one query more than 2^26 below its
largest are rounded, and the largest may not pass 2^105.

Positions are device arrays (int32 or int64, one for each request or one for all), so every call can be captured
in a CUDA graph and replayed as they advance.  Forward only; everything runs on the current CUDA stream.
"""
from __future__ import annotations

import torch

from . import _lib
from .geometry import D, HKV
from .rotary import (_call, _CODE, _current_device, _current_stream, _device_of, _index, _like, _no_grad, _own_rows, _rows,
                     _same_device, _table, _weights)

REC = 144


def new_cache(B, Lmax, dev, hkv=HKV):
    """(B, hkv, Lmax, 144) uint8 records; all zero, which reads as zeros."""
    return torch.zeros(B, hkv, Lmax, REC, dtype=torch.uint8, device=dev)


def _cache(cache, ndim=4):
    """The block's fields of a cache; sizes and strides are checked by the entry."""
    if not isinstance(cache, torch.Tensor) or not cache.is_cuda or cache.dtype is not torch.uint8 or cache.dim() != ndim:
        if not isinstance(cache, torch.Tensor) or not cache.is_cuda:
            raise RuntimeError("cache must be a CUDA tensor")
        raise RuntimeError(f"cache must be {'(B, hkv, Lmax, 144)' if ndim == 4 else '(B * hkv, Lmax, 144)'} uint8, got "
                           f"{tuple(cache.shape)} {cache.dtype}")
    return cache.data_ptr(), *cache.shape, *cache.stride()


_NO_ROWS = (0,) * 9


def append(cache, k, v, start, *, offset=0, lens=None):
    """Writes k, v (B, hkv, T, 128) bf16 into the cache (B, hkv, Lmax, 144): row i of request b at position
    start[b] + offset + i.  Rows i >= lens[b] (default T) and positions outside [0, Lmax) write nothing.
    Calls that write the same positions must be ordered (one stream, or events)."""
    fc, dev, bf = _cache(cache), cache.get_device(), torch.bfloat16
    _call(dev, "oa_kv4_append", *_NO_ROWS, *_rows("k", k, bf, dev), *_rows("v", v, bf, dev), *_NO_ROWS, *fc, 0, 0, 0, 0, *_index("start", start, dev),
          *_index("lens", lens, dev), 0, 0, offset, _lib.OA_F32, 0, 0.0)


def rope_append(cache, q, k, v, cos, sin, start, *, offset=0, lens=None, q_weight=None, k_weight=None, eps=1e-5,
                q_out=None):
    """rotary.qk_norm_rope and append in one launch: returns the normalised, rotated q (B, HQ, T, 128) bf16 and
    writes the normalised, rotated k (rounded to bf16) and v into the cache.  Arguments as in those two; rows
    whose position is outside the tables or behind lens are padding (no record; q as in qk_norm_rope), rows at
    positions past the cache rotate q and write no record."""
    fc, dev, bf = _cache(cache), cache.get_device(), torch.bfloat16
    fq = _rows("q", q, bf, dev)
    zero = q_out is None
    if zero:
        q_out = _like(q)
        fo = _own_rows(q_out, fq[1:5])
    else:
        fo = _rows("q_out", q_out, bf, dev)
    qp, kp, wd = _weights(q_weight, k_weight, bf, dev)
    _call(dev, "oa_kv4_append", *fq, *_rows("k", k, bf, dev), *_rows("v", v, bf, dev), *fo, *fc, *_table(cos, sin, dev),
          *_index("start", start, dev), *_index("lens", lens, dev), qp, kp, offset, wd, zero, eps)
    return q_out


def unpack(cache, start, T, *, offset=0, lens=None, out_dtype=torch.bfloat16, k_out=None, v_out=None):
    """The values (k, v), each (B, hkv, T, 128) bf16 or fp32, of the records at positions start[b] + offset + i,
    i < T.  Rows i >= lens[b] and positions outside the cache are zero in outputs that this call allocates and
    left as they were in k_out / v_out."""
    fc, dev = _cache(cache), cache.get_device()
    zk, zv = k_out is None, v_out is None
    if not (zk and zv):
        _same_device(dev, k_out=k_out, v_out=v_out)
        out_dtype = (v_out if zk else k_out).dtype
    if T < 0 or out_dtype not in _CODE:
        raise RuntimeError(f"T must be >= 0 and the outputs bf16 or fp32, got {T}, {out_dtype}")
    shape = (fc[1], fc[2], T, D)
    if zk:
        k_out = cache.new_empty(shape, dtype=out_dtype)
        fk = _own_rows(k_out, shape)
    else:
        fk = _rows("k_out", k_out, out_dtype, dev)
        if k_out.shape != shape:
            raise RuntimeError(f"k_out must be {shape}, got {tuple(k_out.shape)}")
    if zv:
        v_out = _like(k_out)
        fv = _own_rows(v_out, shape)
    else:
        fv = _rows("v_out", v_out, out_dtype, dev)
    _call(dev, "oa_kv4_unpack", *fc, *fk, *fv, *_index("start", start, dev), *_index("lens", lens, dev), offset,
          _CODE[out_dtype], zk, zv)
    return k_out, v_out


_ws_cache: dict = {}


def attention_workspace(B, HQ, T, cache_len, dev, hkv=HKV):
    """Scratch of decode_attention (uint8, zero-filled, 2.4 MB and 4 bytes a row) for these sizes and all that have no
    more requests, KV heads and blocks of 8 queries of a KV head.  Calls that can overlap on the GPU must not share
    one."""
    with torch.cuda.device(dev):
        need = _lib.load().oa_kv4_attention_workspace_bytes(B, HQ, hkv, T, cache_len)
    return torch.zeros(max(need, 16), dtype=torch.uint8, device=dev)


def _workspace(dev, *sizes):
    """The kept workspace of a GPU and stream, grown on demand: calls on one stream run in order and may share it.  A
    call that is being captured gets its own from the graph's pool, where its zero-fill is replayed too."""
    if dev == _current_device():
        capturing = torch.cuda.is_current_stream_capturing()
    else:
        with torch.cuda.device(dev):
            capturing = torch.cuda.is_current_stream_capturing()
    key = (dev, _current_stream(dev))
    kept = None if capturing else _ws_cache.get(key)
    if kept is not None and sizes in kept[1]:
        return kept[0]
    with torch.cuda.device(dev):
        need = _lib.load().oa_kv4_attention_workspace_bytes(*sizes)
    if kept is not None and kept[0].numel() >= need:
        if len(kept[1]) < 4096:
            kept[1].add(sizes)
        return kept[0]
    ws = torch.zeros(max(need, 16), dtype=torch.uint8, device=f"cuda:{dev}")
    if not capturing:
        _ws_cache[key] = (ws, {sizes})
    return ws


def decode_attention(q, cache, n, *, offset=0, sm_scale=None, out_dtype=None, out=None, workspace=None):
    """q (B, HQ, T, 128) bf16 over the cache (B, hkv, Lmax, 144) -> (B, HQ, T, 128) in out_dtype (bf16, the
    default, or fp32; either holds about 11 bits of the codes' part, see above).

    n (B,) or (1,) int32 or int64 on the device: request b's length is min(n[b] + offset, Lmax), its T query
    tokens the last T positions; token i sees positions <= length - T + i.  HQ is a multiple of hkv, query head h
    reads KV head h // (HQ // hkv).  A query token before the first position (a length below T, zero or
    negative) gives zeros.  Records at positions >= the length are never used.  sm_scale defaults to 128**-0.5.
    out must not overlap q or the cache.

    workspace: attention_workspace(...) of these sizes or larger ones.  By default one is kept for each device and
    stream; a call that is being captured allocates its own from the graph's pool (graphs may then be replayed
    side by side), so a decode loop that captures many layers passes one."""
    dev, fc = _device_of("q", q), _cache(cache)
    fq = _rows("q", q, torch.bfloat16, dev)
    if cache.get_device() != dev or workspace is not None or out is not None:
        _same_device(dev, cache=cache, workspace=workspace, out=out)
    dt = torch.bfloat16 if out_dtype is None else out_dtype
    if out is not None and out_dtype is None:
        dt = out.dtype
    if dt not in _CODE or (out is not None and dt != out.dtype):
        raise RuntimeError(f"the output must be bf16 or fp32 and out of type out_dtype, got {dt}"
                           f"{'' if out is None else f' and out {out.dtype}'}")
    if out is None:
        out = _like(q) if out_dtype is None else q.new_empty(fq[1:5], dtype=dt)
        fo = _own_rows(out, fq[1:5])
    else:
        fo = _rows("out", out, dt, dev)
    if workspace is None:
        workspace = _workspace(dev, *fq[1:3], fc[2], fq[3], fc[3])
    elif workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise RuntimeError("workspace must be a contiguous uint8 tensor")
    _call(dev, "oa_kv4_attention", *fq, *fc, *fo, *_index("n", n, dev), workspace.data_ptr(),
          workspace.numel(), offset, _CODE[dt], D ** -0.5 if sm_scale is None else sm_scale)
    return out


_NO_PROXIES, _NO_LOG = (0,) * 14, (0,) * 5


def _list(t, dev):
    """The block's fields of an index list; None: not one on GPU `dev`."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.dim() != 2 or t.get_device() != dev:
        return None
    return t.data_ptr(), *t.shape, *t.stride()


def flash_attention(q, cache, sel_idx, exp_idx, kbar, vbar, log_n, nb=None, *, sm_scale=None, out_dtype=None,
                    out=None):
    """flash.ours_flash / flash.decode_expand_attention over a 4-bit cache: q (BQ, 128) bf16, cache (BH, Lmax, 144)
    -> (BQ, 128) in out_dtype (bf16 or fp32, with about 11 bits of the codes' part, see above).  Row r reads KV row
    r // (BQ // BH).

    One softmax over the tokens of sel_idx (BQ, n_sel) and exp_idx (BQ, n_exp) (int32; an index outside [0, Lmax)
    is padding) and nb cluster proxies with logits q . kbar * sm_scale + log_n (log_n = -inf skips one).
    kbar, vbar bf16 (BQ, NB, 128) (for each query row) or (BH, NB, 128) (for each KV row), log_n (BQ, NB) fp32;
    nb = 0 disables the proxies.  A token that a row lists twice counts twice.  A row with nothing to attend gives
    zeros.  out must not overlap the inputs."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda or q.dtype is not torch.bfloat16 or q.dim() != 2:
        raise RuntimeError("q must be a (rows, 128) bf16 CUDA tensor")
    _no_grad("q", q)
    fc, dev = _cache(cache, ndim=3), q.get_device()
    fs, fe = _list(sel_idx, dev), _list(exp_idx, dev)
    if fs is None or fe is None or cache.get_device() != dev or out is not None:
        _same_device(dev, cache=cache, sel_idx=sel_idx, exp_idx=exp_idx, out=out)
    if fs is None or fe is None:
        got = " and ".join(f"{tuple(t.shape)} {t.dtype}" if isinstance(t, torch.Tensor) else type(t).__name__
                           for t in (sel_idx, exp_idx))
        raise RuntimeError(f"sel_idx and exp_idx must be (rows, n) int32 tensors, got {got}")
    NB = (0 if kbar is None else kbar.shape[1]) if nb is None else int(nb)
    fb, fl = _NO_PROXIES, _NO_LOG
    if NB > 0:
        if kbar is None or vbar is None or log_n is None or kbar.dtype is not torch.bfloat16 or kbar.dim() != 3 or \
                vbar.dtype is not torch.bfloat16 or vbar.dim() != 3 or log_n.dtype is not torch.float32 or log_n.dim() != 2:
            raise RuntimeError("kbar and vbar must be (rows, NB, 128) bf16 and log_n (rows, NB) fp32")
        if not kbar.get_device() == vbar.get_device() == log_n.get_device() == dev:
            _same_device(dev, kbar=kbar, vbar=vbar, log_n=log_n)
        for name, t in (("kbar", kbar), ("vbar", vbar), ("log_n", log_n)):
            _no_grad(name, t)
        fb = (kbar.data_ptr(), *kbar.shape, *kbar.stride(), vbar.data_ptr(), *vbar.shape, *vbar.stride())
        fl = (log_n.data_ptr(), *log_n.shape, *log_n.stride())
    if out is None:
        out = _like(q) if out_dtype is None else q.new_empty(q.shape, dtype=out_dtype)
    dt = out.dtype
    if dt not in _CODE or out.dim() != 2 or (out_dtype is not None and out_dtype != dt):
        raise RuntimeError(f"out must be (rows, 128) bf16 or fp32 of type out_dtype, got {tuple(out.shape)} {dt}")
    _call(dev, "oa_kv4_flash", q.data_ptr(), *q.shape, *q.stride(), *fc, *fs, *fe, *fb, *fl, out.data_ptr(),
          *out.shape, *out.stride(), _CODE[dt], NB, D ** -0.5 if sm_scale is None else sm_scale)
    return out
