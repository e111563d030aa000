"""Cases of the 4-bit K/V cache operators and of the query/key rotation that feeds them.

    rope     rotary.qk_norm_rope: optional per-head RMS norm of q and k, then the position rotation
    write    kv4.append, read back with kv4.unpack: rows enter the 4-bit cache and leave it as values
    step     kv4.rope_append, read back with kv4.unpack: one decode step's rotation and cache write
    dense    kv4.decode_attention: every query row attends to all positions of its request
    lists    kv4.flash_attention: every query row attends to its index lists and cluster proxies

A cache record holds one token of one KV head in 144 bytes: 64 bytes of K codes, 64 bytes of V codes, and
eight bf16 numbers (scale, offset) of K's first and second half and of V's.  Byte j of a 64-byte block holds
the code of dimension j in its low nibble and of dimension j + 64 in its high one; a value is
scale * code + offset.
"""
import math
import random

import numpy as np
import torch

own = False

D = 128
REC = 144
DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 32 requests: q and k are slices of the fused projection's rows
        dict(name="rope decode 32", op="rope", B=32, T=1, HQ=32, HKV=8, R=128, norm=False, f32=False, ragged=False,
             at=32768),
        # an ordinary prompt, keys and queries normalised per head
        dict(name="rope prompt 8191 norm", op="rope", B=1, T=8191, HQ=32, HKV=8, R=128, norm=True, f32=False,
             ragged=False, at=0),
        # a padded batch in fp32 with half of each head rotated
        dict(name="rope padded fp32", op="rope", B=3, T=1021, HQ=8, HKV=2, R=64, norm=True, f32=True, ragged=True,
             at=17),
        # a prompt enters the cache
        dict(name="write prompt 8192", op="write", B=1, T=8192, HKV=8, ragged=False, at=0),
        # short ragged continuations enter at different positions
        dict(name="write ragged 37", op="write", B=16, T=37, HKV=8, ragged=True, at=1000),
        # what one decode step of 32 requests does before its attention
        dict(name="step 32", op="step", B=32, T=1, HQ=32, HKV=8, R=128, ragged=False, at=4095),
        # first tokens after a short prompt, one request: latency
        dict(name="dense 1x129", op="dense", B=1, HQ=32, HKV=8, T=1, n=129, cap=512, mix=0),
        # one request with a long context
        dict(name="dense 1x32768", op="dense", B=1, HQ=32, HKV=8, T=1, n=32768, cap=32784, mix=0),
        # a serving batch of requests of mixed age, two query tokens each (a drafted token is verified)
        dict(name="dense 64 ragged", op="dense", B=64, HQ=32, HKV=8, T=2, n=8191, cap=8200, mix=5),
        # the benchmark's batch and context
        dict(name="dense 32x32768", op="dense", B=32, HQ=32, HKV=8, T=1, n=32768, cap=32784, mix=0),
        # the benchmark's 1% read: 15 selected, 216 expanded, 64 clusters
        dict(name="lists 32 at 1%", op="lists", B=32, HQ=32, HKV=8, n=32768, sel=15, exp=216, nb=64),
        # one request at the 5% read
        dict(name="lists 1 at 5%", op="lists", B=1, HQ=32, HKV=8, n=32768, sel=15, exp=1335, nb=192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "write", "step", "dense", "dense", "lists"])
    hkv = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 4, 4, 7, 8])
    if op == "rope":
        B = _log(rng, 1, 48)
        T = _log(rng, 1, max(1, 16384 // B))
        return dict(op=op, B=B, T=T, HQ=hkv * g, HKV=hkv, R=rng.choice([32, 64, 96, 128]), norm=rng.random() < 0.5,
                    f32=rng.random() < 0.3, ragged=rng.random() < 0.5, at=rng.randrange(0, 20000))
    if op == "write":
        B = _log(rng, 1, 48)
        return dict(op=op, B=B, T=_log(rng, 1, max(1, 16384 // B)), HKV=hkv, ragged=rng.random() < 0.5,
                    at=rng.randrange(0, 3000))
    if op == "step":
        return dict(op=op, B=_log(rng, 1, 256), T=rng.choice([1, 1, 2, 3]), HQ=hkv * g, HKV=hkv,
                    R=rng.choice([64, 128]), ragged=False, at=rng.randrange(0, 5000))
    if op == "dense":
        B = _log(rng, 1, 128)
        n = _log(rng, 1, max(2, min(100000, 400000 // B)))
        return dict(op=op, B=B, HQ=hkv * g, HKV=hkv, T=rng.choice([1, 1, 1, 2, 4]), n=n, cap=n + rng.randrange(0, 40),
                    mix=rng.choice([0, rng.randrange(1, 1000)]))
    n = _log(rng, 64, 32768)
    return dict(op=op, B=_log(rng, 1, 24), HQ=hkv * g, HKV=hkv, n=n, sel=rng.randrange(2, 40),
                exp=min(n, _log(rng, 1, 1500)), nb=rng.choice([0, 16, 64, 192]))


def _lens(case):
    """Rows (or positions) of each request, from the case alone."""
    B = case["B"]
    if case["op"] == "dense":
        if not case["mix"]:
            return [case["n"]] * B
        r = random.Random(case["mix"])
        return [max(1, _log(r, 1, case["n"])) if r.random() < 0.7 else case["n"] for _ in range(B)]
    if not case["ragged"]:
        return [case["T"]] * B
    r = random.Random(B * 1000003 + case["T"])
    return [r.randrange(1, case["T"] + 1) for _ in range(B)]


def _starts(case):
    r = random.Random(case["at"] + case["B"])
    return [case["at"] + (r.randrange(0, 64) if case["ragged"] else 0) for _ in range(case["B"])]


# ------------------------------------------------------------------ inputs
def _table(P, R):
    """cos and sin of every position (P, R): the frequencies are repeated for the two halves."""
    inv = 1.0 / (500000.0 ** (torch.arange(0, R, 2, device=DEV).float() / R))
    f = torch.arange(P, device=DEV).float()[:, None] * inv[None]
    f = torch.cat([f, f], -1)
    return f.cos(), f.sin()


def _rand_cache(B, HKV, n, cap, gen):
    """Records of n Gaussian tokens (keys with a bias for each channel), made by the quantiser below."""
    cache = torch.zeros(B, HKV, cap, REC, dtype=torch.uint8, device=DEV)
    bias = torch.randn(HKV, 1, D, generator=gen, device=DEV) * 1.5
    for b in range(B):
        k = torch.randn(HKV, n, D, generator=gen, device=DEV) + bias
        v = torch.randn(HKV, n, D, generator=gen, device=DEV)
        for x, at, meta in ((k, 0, 128), (v, 64, 136)):
            c, s, z = _quantise(x.bfloat16().float())
            c = c.to(torch.uint8)
            cache[b, :, :n, at:at + 64] = c[..., 0, :] | (c[..., 1, :] << 4)
            m = torch.stack([s[..., 0, 0], z[..., 0, 0], s[..., 1, 0], z[..., 1, 0]], -1).bfloat16()
            cache[b, :, :n, meta:meta + 8] = m.view(torch.uint8)
    return cache


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    B, HKV, op = case["B"], case["HKV"], case["op"]
    HQ = case.get("HQ", HKV)
    s = {"case": case, "op": op}

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    if op in ("rope", "write", "step"):
        T = case["T"]
        dt = torch.float32 if case.get("f32") else torch.bfloat16
        # rows of the fused projection: q heads, k heads, v heads
        qkv = torch.randn(B, T, (HQ + 2 * HKV) * D, generator=g, device=DEV)
        qkv[..., HQ * D:(HQ + HKV) * D] += torch.randn(HKV * D, generator=g, device=DEV)
        s["qkv"] = qkv.to(dt)
        s["start"] = i32(_starts(case))
        s["lens"] = i32(_lens(case)) if case["ragged"] else None
        P = max(_starts(case)) + T
        if op != "write":
            s["cos"], s["sin"] = _table(P, case["R"])
        s["wq"] = s["wk"] = None
        if case.get("norm"):
            s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(dt) for _ in range(2))
        if op != "rope":
            s["cache"] = torch.zeros(B, HKV, P, REC, dtype=torch.uint8, device=DEV)
    elif op == "dense":
        s["cache"] = _rand_cache(B, HKV, case["n"], case["cap"], g)
        s["q"] = torch.randn(B, HQ, case["T"], D, generator=g, device=DEV).bfloat16()
        s["n"] = i32(_lens(case))
    else:
        n, R, nb = case["n"], B * HQ, case["nb"]
        s["cache"] = _rand_cache(B, HKV, n, n, g).view(B * HKV, n, REC)
        s["q"] = torch.randn(R, D, generator=g, device=DEV).bfloat16()
        pick = torch.rand(R, n, generator=g, device=DEV).argsort(-1)[:, :case["sel"] + case["exp"]].int()
        if pick.shape[1] < case["sel"] + case["exp"]:  # fewer positions than entries: the rest is padding
            pick = torch.nn.functional.pad(pick, (0, case["sel"] + case["exp"] - pick.shape[1]), value=-1)
        s["sel"] = pick[:, :case["sel"]].contiguous()
        s["exp"] = pick[:, case["sel"]:].contiguous()
        s["exp"][:, case["exp"] - case["exp"] // 16:] = -1  # lists that were not filled
        s["kbar"] = torch.randn(R, nb, D, generator=g, device=DEV).bfloat16()
        s["vbar"] = (torch.randn(R, nb, D, generator=g, device=DEV) * 0.3).bfloat16()
        ln = (torch.rand(R, nb, generator=g, device=DEV) * 600 + 1).log()
        if nb:  # one bin in eight was read in full
            dead = torch.rand(R, nb, generator=g, device=DEV).argsort(-1)[:, :nb // 8]
            ln.scatter_(1, dead, -math.inf)
        s["log_n"] = ln
    return s


# ------------------------------------------------------------------ plain forms (32 bits)
def _slices(s):
    c = s["case"]
    B, T, HKV = c["B"], c["T"], c["HKV"]
    HQ = c.get("HQ", HKV)
    x = s["qkv"]
    q = x[..., :HQ * D].view(B, T, HQ, D).transpose(1, 2)
    k = x[..., HQ * D:(HQ + HKV) * D].view(B, T, HKV, D).transpose(1, 2)
    v = x[..., (HQ + HKV) * D:].view(B, T, HKV, D).transpose(1, 2)
    return q, k, v


def _valid(s, T):
    """(B, 1, T, 1): rows that are no padding."""
    i = torch.arange(T, device=DEV)
    n = s["lens"] if s["lens"] is not None else torch.full_like(s["start"], T)
    return (i[None] < n[:, None])[:, None, :, None]


def _rope(s, x, w):
    """x (B, H, T, 128): norm, rotation, one rounding; padded rows are zero."""
    T, R = x.shape[2], s["cos"].shape[1]
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-5) * w.float()
    p = s["start"].long()[:, None] + torch.arange(T, device=DEV)
    cos, sin = s["cos"][p][:, None], s["sin"][p][:, None]
    a, rest = y[..., :R], y[..., R:]
    rot = torch.cat([-a[..., R // 2:], a[..., :R // 2]], -1)
    y = torch.cat([a * cos + rot * sin, rest], -1)
    return torch.where(_valid(s, T), y, torch.zeros_like(y)).to(x.dtype)


def _quantise(x):
    """x (..., 128) fp32 -> codes (..., 2, 64), scale and offset (..., 2, 1), all fp32."""
    x = x.reshape(*x.shape[:-1], 2, 64)
    z = x.amin(-1, keepdim=True)
    sc = ((x.amax(-1, keepdim=True) - z) / 15.0).bfloat16().float()
    c = (x - z) / torch.where(sc > 0, sc, torch.ones_like(sc))
    return c.round().clamp(0, 15), sc, z  # ties go to the even code


def _round_trip(s, x):
    c, sc, z = _quantise(x.float())
    y = (sc * c + z).flatten(-2)
    return torch.where(_valid(s, x.shape[2]), y, torch.zeros_like(y)).bfloat16()


def _values(rec, at, meta):
    """Values of one side (K: 0, 128; V: 64, 136) of records (..., 144), fp32 (..., 128)."""
    byte = rec[..., at:at + 64]
    m = rec[..., meta:meta + 8].contiguous().view(torch.bfloat16).float()
    lo = (byte & 15).float() * m[..., 0:1] + m[..., 1:2]
    hi = (byte >> 4).float() * m[..., 2:3] + m[..., 3:4]
    return torch.cat([lo, hi], -1)


def _attend(z, v):
    """softmax(z) v over the last axis of z; a row of -inf gives zeros."""
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = (z - m).exp()
    den = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(den == 0, torch.ones_like(den), den)


def _dense(s):
    c = s["case"]
    B, HKV, T, n = c["B"], c["HKV"], c["T"], c["n"]
    rec = s["cache"][:, :, :n]
    q = s["q"].float().reshape(B, HKV, -1, D)  # rows (head of the group, query token)
    z = (q @ _values(rec, 0, 128).transpose(-1, -2)) * D ** -0.5
    last = s["n"].long()[:, None] - T + torch.arange(T, device=DEV)  # a query token's own position
    ok = torch.arange(n, device=DEV) <= last[..., None]  # (B, T, n)
    ok = ok[:, None, None].expand(B, HKV, c["HQ"] // HKV, T, n).reshape(z.shape)
    z = torch.where(ok, z, torch.full_like(z, -math.inf))
    return _attend(z, _values(rec, 64, 136)).view(B, c["HQ"], T, D).bfloat16()


def _lists(s):
    c = s["case"]
    kv = torch.arange(s["q"].shape[0], device=DEV) // (c["HQ"] // c["HKV"])
    idx = torch.cat([s["sel"], s["exp"]], 1).long()
    rec = s["cache"][kv[:, None], idx.clamp(min=0)]  # (R, entries, 144)
    q = s["q"].float()[:, None]
    z = (q @ _values(rec, 0, 128).transpose(-1, -2)) * D ** -0.5
    z = torch.where((idx >= 0)[:, None], z, torch.full_like(z, -math.inf))
    zp = (q @ s["kbar"].float().transpose(-1, -2)) * D ** -0.5 + s["log_n"][:, None]
    v = torch.cat([_values(rec, 64, 136), s["vbar"].float()], 1)
    return _attend(torch.cat([z, zp], -1), v)[:, 0].bfloat16()


def run(state):
    s, op = state, state["op"]
    if op in ("rope", "write", "step"):
        q, k, v = _slices(s)
        T = s["case"]["T"]
    if own:
        from openattention_b200 import kv4, rotary
        if op == "rope":
            return rotary.qk_norm_rope(q, k, s["cos"], s["sin"], s["start"], lens=s["lens"], q_weight=s["wq"],
                                       k_weight=s["wk"], eps=1e-5)
        if op == "write":
            kv4.append(s["cache"], k, v, s["start"], lens=s["lens"])
            return kv4.unpack(s["cache"], s["start"], T, lens=s["lens"])
        if op == "step":
            qr = kv4.rope_append(s["cache"], q, k, v, s["cos"], s["sin"], s["start"], lens=s["lens"])
            return (qr, *kv4.unpack(s["cache"], s["start"], T, lens=s["lens"]))
        if op == "dense":
            return kv4.decode_attention(s["q"], s["cache"], s["n"])
        return kv4.flash_attention(s["q"], s["cache"], s["sel"], s["exp"], s["kbar"], s["vbar"], s["log_n"])
    if op == "rope":
        return _rope(s, q, s["wq"]), _rope(s, k, s["wk"])
    if op == "write":
        return _round_trip(s, k), _round_trip(s, v)
    if op == "step":
        return _rope(s, q, None), _round_trip(s, _rope(s, k, None)), _round_trip(s, v)
    return _dense(s) if op == "dense" else _lists(s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op, B, HKV = case["op"], case["B"], case["HKV"]
    HQ = case.get("HQ", HKV)
    if op in ("rope", "write", "step"):
        size = 4 if case.get("f32") else 2
        rows, out_rows = sum(_lens(case)), B * case["T"]
        heads = {"rope": HQ + HKV, "write": 2 * HKV, "step": HQ + 2 * HKV}[op]
        by = rows * heads * D * size + out_rows * heads * D * size
        fl = rows * heads * D * 4
        if op != "write":
            by += len({st + i for st, n in zip(_starts(case), _lens(case)) for i in range(n)}) * 2 * case["R"] * 4
        if op != "rope":
            by += 2 * rows * HKV * REC  # the records are written, and read back
        return {"bytes": by, "flops": fl}
    if op == "dense":
        tok = sum(_lens(case))
        io = 2 * B * HQ * case["T"] * D * 2
        return {"bytes": tok * HKV * REC + io, "flops": 4 * D * HQ * case["T"] * tok}
    R, n = B * HQ, case["n"]
    entries = min(n, case["sel"] + case["exp"] - case["exp"] // 16)
    # a record that several heads of one group list is counted once
    distinct = n * (1 - (1 - entries / n) ** (HQ // HKV))
    live = case["nb"] - case["nb"] // 8
    by = B * HKV * distinct * REC + R * (case["sel"] + case["exp"]) * 4 + R * (live * 2 * D * 2 + case["nb"] * 4)
    return {"bytes": by + 2 * R * D * 2, "flops": 4 * D * R * (entries + live)}


# ------------------------------------------------------------------ the definition in 64 bits
def _rope64(x, w, cos, sin, start, lens):
    """One array (B, H, T, 128) in float64, request by request and by complex rotation of the pairs."""
    x = x.double()
    out = torch.zeros_like(x)
    h = cos.shape[1] // 2
    c, sn = cos.double(), sin.double()
    for b, (p, n) in enumerate(zip(start, lens)):
        y = x[b, :, :n]
        if w is not None:
            y = y * w.double() / torch.sqrt(y.square().sum(-1, keepdim=True) / D + 1e-5)
        u, v = y[..., :h], y[..., h:2 * h]
        out[b, :, :n, :h] = u * c[p:p + n, :h] - v * sn[p:p + n, :h]
        out[b, :, :n, h:2 * h] = v * c[p:p + n, h:] + u * sn[p:p + n, h:]
        out[b, :, :n, 2 * h:] = y[..., 2 * h:]
    return out


def _trip64(x, lens):
    """The stored value of every element: the nearest of the group's sixteen levels, by index arithmetic."""
    x = x.double()
    out = torch.zeros_like(x)
    for b, n in enumerate(lens):
        for half in (slice(0, 64), slice(64, 128)):
            y = x[b, :, :n, half]
            lo, hi = torch.aminmax(y, dim=-1, keepdim=True)
            step = ((hi - lo) / 15).to(torch.bfloat16).double()
            i = torch.round((y - lo) / torch.where(step == 0, torch.ones_like(step), step))
            out[b, :, :n, half] = lo + step * torch.clamp(i, max=15)
    return out


_NIBBLE = np.stack([np.arange(256) % 16, np.arange(256) // 16], -1)


def _values64(rec, side):
    """Values (n, 128) of side 0 (K) or 1 (V) of records (n, 144), by a table of the 256 bytes."""
    table = torch.from_numpy(_NIBBLE).to(rec.device).double()
    code = table[rec[:, 64 * side:64 * side + 64].long()].permute(0, 2, 1)  # (n, half, 64)
    raw = rec[:, 128 + 8 * side:136 + 8 * side].long()
    bits = (raw[:, 0::2] + 256 * raw[:, 1::2]).int() * 65536
    m = bits.view(torch.float32).double().view(-1, 2, 2)
    return (code * m[..., :1] + m[..., 1:]).reshape(-1, D)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("rope", "write", "step"):
        q, k, v = _slices(s)
        st, n = _starts(case), _lens(case)
    if op == "rope":
        return tuple(_rope64(x, w, s["cos"], s["sin"], st, n) for x, w in ((q, s["wq"]), (k, s["wk"])))
    if op == "write":
        return _trip64(k, n), _trip64(v, n)
    if op == "step":
        q, k = (_rope64(x, None, s["cos"], s["sin"], st, n) for x in (q, k))
        return q, _trip64(k.to(torch.bfloat16), n), _trip64(v, n)  # a rotated key is a bf16 row
    B, HKV, HQ = case["B"], case["HKV"], case["HQ"]
    G = HQ // HKV
    if op == "dense":
        T = case["T"]
        out = torch.zeros(B, HQ, T, D, dtype=torch.float64, device=DEV)
        for b, n in enumerate(_lens(case)):
            for h in range(HKV):
                K, V = (_values64(s["cache"][b, h, :n], side) for side in (0, 1))
                for t in range(T):
                    m = n - T + 1 + t
                    if m > 0:
                        q = s["q"][b, h * G:(h + 1) * G, t].double()
                        out[b, h * G:(h + 1) * G, t] = torch.softmax(q @ K[:m].T / math.sqrt(D), -1) @ V[:m]
        return out
    R = B * HQ
    out = torch.zeros(R, D, dtype=torch.float64, device=DEV)
    idx = torch.cat([s["sel"], s["exp"]], 1)
    for r in range(R):
        i = idx[r][idx[r] >= 0].long()
        rec = s["cache"][r // G, i]
        K = torch.cat([_values64(rec, 0), s["kbar"][r].double()])
        V = torch.cat([_values64(rec, 1), s["vbar"][r].double()])
        z = K @ s["q"][r].double() / math.sqrt(D)
        z[len(i):] += s["log_n"][r].double()
        out[r] = torch.softmax(z, 0) @ V
    return out
