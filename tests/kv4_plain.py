"""The rotation's, the 4-bit cache's and its attentions' definitions in 64 bits (CPU), and what a right kernel
may be off by.  A rounding to bf16 is off by at most 2^-8 of the value, to fp16 2^-11, to fp32 2^-24."""
import math

import torch

D, REC = 128, 144


def table(P, R, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(P, R, generator=g) * 6.28  # the halves differ: every entry of the table counts
    return a.cos(), a.sin()


def rope(x, cos, sin, start, lens, w=None, eps=1e-5):
    """(value, slack) in fp64 for x (B, H, T, 128); rows that are padding are zero.

    slack: the fp32 arithmetic before the last rounding.  The norm's sum of 128 squares (8 in a lane, 4
    shuffles: 12 roundings on the longest path, halved by the root), mean, eps, root (2 ulp) and two products:
    under 16 steps of 2^-24; the rotation's products and sum: 3.  32 covers both."""
    x = x.double()
    B, H, T, _ = x.shape
    P, R = cos.shape
    h = R // 2
    out, slack = torch.zeros_like(x), torch.zeros_like(x)
    for b in range(B):
        for t in range(T):
            p = start[b] + t
            if t >= lens[b] or p < 0 or p >= P:
                continue
            y = x[b, :, t]
            if w is not None:
                y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
            c, s = cos[p].double(), sin[p].double()
            rot = torch.cat([-y[:, h:R], y[:, :h]], -1)
            out[b, :, t] = y
            out[b, :, t, :R] = y[:, :R] * c + rot * s
            slack[b, :, t] = y.abs()
            slack[b, :, t, :R] = (y[:, :R] * c).abs() + (rot * s).abs()
    return out, slack * 32 * 2.0 ** -24


def quantise(x):
    """x (..., 128) bf16 -> records' parts: codes (..., 128) int, scale, offset (..., 2) fp32.  The scale is
    defined by fp32 operations (one subtraction, one division, one rounding to bf16)."""
    g = x.float().unflatten(-1, (2, 64))
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / 15).bfloat16().float()
    bad = ~torch.isfinite(g).all(-1) | ~torch.isfinite(hi - lo)
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    lo = torch.where(bad, torch.zeros_like(lo), lo)
    q = (g.double() - lo.double()[..., None]) / torch.where(s > 0, s, torch.ones_like(s)).double()[..., None]
    code = torch.where((s > 0)[..., None], q.round().clamp(0, 15), torch.zeros_like(q))
    return code.nan_to_num(0).flatten(-2).int(), s, lo


def pack(k, v):
    """Records (..., 144) uint8 of bf16 rows (..., 128)."""
    parts, meta = [], []
    for x in (k, v):
        c, s, z = quantise(x)
        parts.append((c[..., :64] | (c[..., 64:] << 4)).to(torch.uint8))
        meta.append(torch.stack([s[..., 0], z[..., 0], s[..., 1], z[..., 1]], -1).bfloat16())
    return torch.cat(parts + [torch.cat(meta, -1).contiguous().view(torch.uint8)], -1)


def parts(rec, side):
    """(codes, scale, offset), each (..., 128) fp64, of one side of records."""
    b = rec[..., 64 * side:64 * side + 64]
    code = torch.cat([b & 15, b >> 4], -1).double()
    m = rec[..., 128 + 8 * side:136 + 8 * side].contiguous().view(torch.bfloat16).double()
    s = torch.cat([m[..., 0:1].expand_as(code[..., :64]), m[..., 2:3].expand_as(code[..., :64])], -1)
    z = torch.cat([m[..., 1:2].expand_as(code[..., :64]), m[..., 3:4].expand_as(code[..., :64])], -1)
    return code, s, z


def values(rec, side):
    c, s, z = parts(rec, side)
    return s * c + z


def attend(q, rec, scale, kbar=None, vbar=None, log_n=None):
    """(out, slack) for one query row q (128,) over records rec (n, 144) and proxies.

    slack, before the last rounding.  Logits: q . k is a sum of 128 products s * code * q and z * q in fp32,
    off by at most 2^-16 of the sum of their magnitudes (256 roundings); a logit off by e moves a weight by
    2e at most, so the row by 2e times the magnitudes it sums.  Values: weight * scale is rounded to fp16
    (2^-11), its product with a code is exact; the offsets' part and the proxies' stay in fp32."""
    ck, sk, zk = parts(rec, 0)
    cv, sv, zv = parts(rec, 1)
    q = q.double()
    z = (sk * ck + zk) @ q * scale
    mag = (sk * ck + zk.abs()) @ q.abs() * abs(scale)
    v, cod = sv * cv + zv, sv * cv
    if kbar is not None and kbar.shape[0]:
        z = torch.cat([z, kbar.double() @ q * scale + log_n.double()])
        mag = torch.cat([mag, kbar.double().abs() @ q.abs() * abs(scale) + log_n.double().abs().nan_to_num(posinf=0)])
        v = torch.cat([v, vbar.double()])
        cod = torch.cat([cod, torch.zeros_like(vbar.double())])
    live = z > -math.inf
    if not live.any():
        return torch.zeros(D, dtype=torch.float64), torch.zeros(D, dtype=torch.float64)
    z, mag, v, cod = z[live], mag[live], v[live], cod[live]
    w = torch.softmax(z, 0)
    e = 2.0 ** -16 * mag.max() + 2.0 ** -20
    return w @ v, 2.0 ** -11 * (w @ cod) + 2 * e * (w @ (cod + v.abs())) + 1e-37


def check(got, want, slack, what=""):
    """got (bf16 or fp32) within its rounding of want (fp64) plus slack."""
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - (half * (want.abs() + slack) + slack)
    assert over.max().item() <= 0, f"{what}: off by {over.max().item():.3e} more than rounding allows"
