"""rotary.qk_norm_rope and the 4-bit cache (append, rope_append, unpack, decode_attention, flash_attention) on
the GPU against their definitions in 64 bits (kv4_plain.py, which derives the tolerances)."""
import math

import pytest
import torch

import kv4_plain as P
from openattention_b200 import kv4, rotary

pytestmark = pytest.mark.gpu
D, REC = 128, 144
BF = torch.bfloat16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(g, *shape, dtype=BF):
    return (torch.randn(*shape, generator=g) * 2 + torch.randn(D, generator=g)).to(dtype)


def _records(g, *lead):
    return P.pack(_rows(g, *lead, D), _rows(g, *lead, D))


# ------------------------------------------------------------------ rotation
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("B,T,HQ,HKV,R,norm", [(1, 1, 32, 8, 128, False), (3, 5, 7, 1, 64, True), (2, 33, 8, 2, 16, True),
                                               (40, 1, 4, 4, 96, True), (1, 700, 32, 8, 128, True)])
def test_qk_norm_rope(B, T, HQ, HKV, R, norm, dtype):
    g = _gen(B * 31 + T)
    tab = 64 + T
    cos, sin = P.table(tab, R)
    q, k = _rows(g, B, HQ, T, D, dtype=dtype), _rows(g, B, HKV, T, D, dtype=dtype)
    wq, wk = ((torch.randn(D, generator=g) + 1).to(dtype) for _ in range(2)) if norm else (None, None)
    start = torch.randint(-2, 70, (B,), generator=g)  # some rows stand before or behind the table
    lens = torch.randint(0, T + 2, (B,), generator=g)
    out = rotary.qk_norm_rope(q.cuda(), k.cuda(), cos.cuda(), sin.cuda(), start.cuda(), lens=lens.int().cuda(),
                              q_weight=None if wq is None else wq.cuda(), k_weight=None if wk is None else wk.cuda())
    for got, x, w in ((out[0], q, wq), (out[1], k, wk)):
        P.check(got, *P.rope(x, cos, sin, start.tolist(), lens.tolist(), w))


def test_rope_strided_in_place_and_padding_kept():
    """q and k as slices of the fused projection, rotated in place with one start for all; padding rows keep
    their contents in given outputs."""
    g = _gen(5)
    B, T, HQ, HKV = 2, 9, 6, 3
    cos, sin = P.table(40, 128)
    qkv = _rows(g, B, T, (HQ + 2 * HKV), D).cuda()
    x = qkv.transpose(1, 2)
    q, k, v = x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:]
    before = qkv.clone()
    start = torch.tensor([4], device="cuda")
    lens = torch.tensor([9, 6], dtype=torch.int32, device="cuda")
    r = rotary.qk_norm_rope(q, k, cos.cuda(), sin.cuda(), start, offset=-1, lens=lens, q_out=q, k_out=k)
    assert r[0] is q and r[1] is k
    old = before.transpose(1, 2)
    assert torch.equal(v, old[:, HQ + HKV:])
    assert torch.equal(x[1, :, 6:], old[1, :, 6:])
    want, slack = P.rope(old[:, :HQ + HKV].cpu(), cos, sin, [3, 3], [9, 6])
    want[1, :, 6:] = old[1, :HQ + HKV, 6:].cpu().double()
    P.check(x[:, :HQ + HKV], want, slack)


def test_rope_keeps_the_eager_expressions_bits():
    """bf16 rows without a norm: bit for bit the eager x * cos + rotate(x) * sin in fp32, rounded once."""
    g = _gen(6)
    cos, sin = (t.cuda() for t in P.table(300, 128))
    x = _rows(g, 1, 8, 300, D).cuda()
    q, k = rotary.qk_norm_rope(x, x[:, :2], cos, sin, torch.zeros(1, dtype=torch.int32, device="cuda"))
    f = x.float()
    want = (f * cos + torch.cat([-f[..., 64:], f[..., :64]], -1) * sin).to(BF)
    assert torch.equal(q, want) and torch.equal(k, want[:, :2])


# ------------------------------------------------------------------ cache write and read-back
@pytest.mark.parametrize("B,T,hkv", [(1, 1, 8), (2, 7, 3), (33, 2, 1), (1, 1500, 8)])
def test_append_and_unpack(B, T, hkv):
    g = _gen(B + T)
    Lmax = T + 40
    k, v = _rows(g, B, hkv, T, D), _rows(g, B, hkv, T, D)
    k[0, 0, 0] = 3.0                      # a constant group: scale 0
    v[0, 0, 0, :64] *= 1e-38 * 0.01       # a range whose scale is subnormal
    v[0, 0, T - 1, 64:] *= 1e30
    start = torch.randint(-1, 42, (B,), generator=g)
    start[0] = 3
    lens = torch.randint(0, T + 1, (B,), generator=g)
    lens[0] = T
    cache = torch.randint(0, 256, (B, hkv, Lmax, REC), generator=g).to(torch.uint8)
    want = cache.clone()
    rec = P.pack(k, v)
    for b in range(B):
        for t in range(int(lens[b])):
            p = int(start[b]) + t
            if 0 <= p < Lmax:
                want[b, :, p] = rec[b, :, t]
    dev = cache.cuda()
    kv4.append(dev, k.cuda(), v.cuda(), start.cuda(), lens=lens.cuda())
    assert torch.equal(dev.cpu(), want)   # every byte, those of untouched records among them
    for dt in (BF, torch.float32):
        ko, vo = kv4.unpack(dev, start.int().cuda(), T, lens=lens.cuda(), out_dtype=dt)
        for got, side in ((ko, 0), (vo, 1)):
            for b in range(B):
                for t in range(T):
                    p = int(start[b]) + t
                    if t < int(lens[b]) and 0 <= p < Lmax:
                        c, s, z = P.parts(want[b, :, p], side)
                        # scale * code is exact in fp32, so the value is one fp32 sum, then the output's rounding
                        val = (s * c).float() + z.float()
                        assert torch.equal(got[b, :, t].cpu(), val.to(dt))
                    else:
                        assert not got[b, :, t].any()


def test_append_error_is_half_a_step():
    g = _gen(11)
    k, v = _rows(g, 1, 2, 64, D), _rows(g, 1, 2, 64, D)
    cache = kv4.new_cache(1, 64, "cuda", hkv=2)
    start = torch.zeros(1, dtype=torch.int64, device="cuda")
    kv4.append(cache, k.cuda(), v.cuda(), start)
    for got, x, side in zip(kv4.unpack(cache, start, 64, out_dtype=torch.float32), (k, v), (0, 1)):
        _, s, z = P.parts(cache.cpu(), side)
        # half a scale; the top level may fall short by 15 roundings of the scale (2^-9 each) -- less; 2^-23 fp32
        assert ((got.cpu().double() - x.double()).abs() <= s / 2 + 2.0 ** -22 * (z.abs() + 16 * s)).all()


def test_append_nonfinite_rows_read_as_nan():
    g = _gen(12)
    k, v = _rows(g, 1, 1, 4, D), _rows(g, 1, 1, 4, D)
    k[0, 0, 0, 5], k[0, 0, 1, 70], v[0, 0, 2, 3], v[0, 0, 3, 100] = math.nan, math.inf, -math.inf, math.nan
    v[0, 0, 1, 0], v[0, 0, 1, 1] = 3.0e38, -3.0e38   # finite, but their range is not
    cache = kv4.new_cache(1, 4, "cuda", hkv=1)
    start = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv4.append(cache, k.cuda(), v.cuda(), start)
    ko, vo = (t.cpu() for t in kv4.unpack(cache, start, 4))
    bad_k, bad_v = ko.isnan()[0, 0], vo.isnan()[0, 0]
    want_k = torch.zeros(4, D, dtype=torch.bool)
    want_k[0, :64] = want_k[1, 64:] = True
    want_v = torch.zeros(4, D, dtype=torch.bool)
    want_v[2, :64] = want_v[3, 64:] = want_v[1, :64] = True
    assert torch.equal(bad_k, want_k) and torch.equal(bad_v, want_v)


@pytest.mark.parametrize("norm", [False, True])
def test_rope_append_is_rope_then_append(norm):
    g = _gen(13)
    B, T, HQ, HKV, Lmax = 3, 4, 10, 2, 24
    cos, sin = (t.cuda() for t in P.table(20, 64))
    x = _rows(g, B, T, HQ + 2 * HKV, D).cuda().transpose(1, 2)
    q, k, v = x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:]
    w = [(torch.randn(D, generator=g) + 1).cuda() for _ in range(2)] if norm else [None, None]
    start = torch.tensor([2, 18, -3], device="cuda")
    lens = torch.tensor([4, 4, 2], device="cuda")
    one, two = kv4.new_cache(B, Lmax, "cuda", hkv=HKV), kv4.new_cache(B, Lmax, "cuda", hkv=HKV)
    q1 = kv4.rope_append(one, q, k, v, cos, sin, start, lens=lens, q_weight=w[0], k_weight=w[1])
    q2, k2 = rotary.qk_norm_rope(q, k, cos, sin, start, lens=lens, q_weight=w[0], k_weight=w[1])
    # positions outside the table are padding for rope_append: append's rows are cut to them
    kv4.append(two, k2, v, start, lens=torch.tensor([4, 2, 2], device="cuda"))
    assert torch.equal(q1, q2) and torch.equal(one, two)
    assert one[0].any() and not one[2].any()


# ------------------------------------------------------------------ dense attention
def _dense_want(q, cache, n, scale):
    B, HQ, T, _ = q.shape
    HKV, Lmax = cache.shape[1], cache.shape[2]
    out = torch.zeros(B, HQ, T, D, dtype=torch.float64)
    slack = torch.zeros_like(out)
    for b in range(B):
        ln = min(int(n[b]), Lmax)
        for h in range(HQ):
            for t in range(T):
                m = max(0, ln - T + 1 + t)
                out[b, h, t], slack[b, h, t] = P.attend(q[b, h, t], cache[b, h // (HQ // HKV), :m], scale)
    return out, slack


@pytest.mark.parametrize("B,HQ,HKV,T,lens,out_dtype", [
    (1, 32, 8, 1, [129], BF), (1, 8, 8, 1, [1], torch.float32), (4, 4, 1, 1, [0, 31, 32, 33], BF),
    (3, 7, 1, 1, [64, 65, 200], torch.float32), (2, 16, 2, 2, [1, 97], BF), (2, 24, 2, 3, [2, 130], torch.float32),
    (1, 32, 1, 5, [77], BF), (5, 2, 2, 1, [-3, 1000, 5, 1201, 256], BF), (1, 12, 4, 4, [2100], BF),
    (1, 4, 2, 1, [9001], torch.float32)])
def test_dense_attention(B, HQ, HKV, T, lens, out_dtype):
    g = _gen(sum(lens) + HQ)
    Lmax = max(1, min(max(lens), 1200) if B > 1 else max(lens))
    cache = _records(g, B, HKV, Lmax)
    q = _rows(g, B, HQ, T, D)
    n = torch.tensor(lens, dtype=torch.int32)
    got = kv4.decode_attention(q.cuda(), cache.cuda(), n.cuda(), out_dtype=out_dtype)
    assert got.dtype == out_dtype and got.shape == q.shape
    P.check(got, *_dense_want(q, cache, lens, D ** -0.5))


def test_dense_masked_records_never_count():
    """Records behind the length hold NaN scales and all-ones bytes; the result does not see them."""
    g = _gen(21)
    cache = _records(g, 3, 2, 100)
    lens = [1, 40, 99]
    clean = cache.clone()
    for b, n in enumerate(lens):
        cache[b, :, n:] = 255
    q = _rows(g, 3, 8, 1, D)
    got = kv4.decode_attention(q.cuda(), cache.cuda(), torch.tensor(lens, device="cuda"))
    P.check(got, *_dense_want(q, clean, lens, D ** -0.5))


def test_dense_nan_record_reaches_its_rows_only():
    g = _gen(22)
    cache = _records(g, 2, 2, 70)
    cache[0, 1, 50, 128:130] = 255       # a NaN K scale
    cache[1, 0, 3, 136:138] = 255        # a NaN V scale (first half)
    q = _rows(g, 2, 4, 1, D)
    got = kv4.decode_attention(q.cuda(), cache.cuda(), torch.tensor([70], device="cuda")).cpu()
    bad = got.isnan()[:, :, 0]
    want = torch.zeros(2, 4, D, dtype=torch.bool)
    want[0, 2:] = True
    want[1, :2, :64] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("qs,ks,vs", [(1.0, 1.0, 1.0), (1e4, 1e-4, 1e-6), (1e-5, 1e4, 1e4), (30.0, 1.0, 1e-30), (1.0, 1e-3, 1e30)])
def test_dense_magnitudes(qs, ks, vs):
    """Queries, keys and values of very different sizes; one value row is 1e4 times the others (the scales of
    one row's groups then span what fp16 holds)."""
    g = _gen(23)
    k, v = _rows(g, 1, 1, 300, D) * ks, _rows(g, 1, 1, 300, D) * vs
    v[0, 0, 150] *= 1e4
    k[0, 0, 150] *= 0.0
    cache = P.pack(k.to(BF), v.to(BF))
    q = (_rows(g, 1, 4, 1, D) * qs).to(BF)
    for out_dtype in (BF, torch.float32):
        got = kv4.decode_attention(q.cuda(), cache.cuda(), torch.tensor([300], device="cuda"), out_dtype=out_dtype)
        P.check(got, *_dense_want(q, cache, [300], D ** -0.5))


def test_dense_views_offset_scale_and_out():
    """A cache slice (other strides), q as a slice of the fused projection, int64 lengths with an offset, a
    scale of the caller's, a strided fp32 output."""
    g = _gen(24)
    big = _records(g, 2, 4, 130)
    cache = big[:, 1:3, :120]
    x = _rows(g, 2, 1, 12, D)
    q = x.transpose(1, 2)[:, 2:8]
    n = torch.tensor([100], dtype=torch.int64)
    buf = torch.full((2, 6, 1, 2 * D), 7.0, device="cuda")
    dev_big = big.cuda()
    got = kv4.decode_attention(x.cuda().transpose(1, 2)[:, 2:8], dev_big[:, 1:3, :120], n.cuda(), offset=13, sm_scale=0.25,
                               out=buf[..., :D])
    assert got.data_ptr() == buf.data_ptr() and (buf[..., D:] == 7).all()
    P.check(got, *_dense_want(q, cache, [113, 113], 0.25))


def test_dense_long_cache_offsets():
    """Byte offsets past 2^32: the last request's records begin 4.5 GB into the cache."""
    g = _gen(25)
    Lmax, n = 1_000_000, 999_999
    cache = torch.zeros(4, 8, Lmax, REC, dtype=torch.uint8, device="cuda")
    tail = _records(g, 8, 600)
    cache[3, :, n - 600:n] = tail.cuda()
    cache[3, :, n:] = 255
    q = _rows(g, 4, 8, 1, D) * 4
    got = kv4.decode_attention(q.cuda(), cache, torch.tensor([1, 0, 3, n], device="cuda")).cpu()
    assert not got[:3].any()
    # the zero records' logits are 0 and their values 0: they only add to the denominator
    for h in range(8):
        K, V = P.values(tail[h], 0), P.values(tail[h], 1)
        z = K @ q[3, h, 0].double() * D ** -0.5
        w = (z - z.max()).exp()
        want = w @ V / (w.sum() + (n - 600) * (-z.max()).exp())
        _, slack = P.attend(q[3, h, 0], tail[h], D ** -0.5)
        P.check(got[3, h, 0], want, slack)
    kv4.append(cache, _rows(g, 4, 8, 1, D).cuda(), _rows(g, 4, 8, 1, D).cuda(), torch.tensor([n], device="cuda"))
    ko, _ = kv4.unpack(cache, torch.tensor([n], device="cuda"), 1)
    assert torch.isfinite(ko).all() and ko[3].any()


def test_dense_repeatable_and_on_other_streams():
    """The same bits from call to call, with calls on two streams at once, and with a caller's workspace."""
    g = _gen(26)
    cache = _records(g, 2, 2, 3000).cuda()
    q = _rows(g, 2, 8, 1, D).cuda()
    n = torch.tensor([2999, 1500], dtype=torch.int32, device="cuda")
    want = kv4.decode_attention(q, cache, n)
    ws = kv4.attention_workspace(2, 8, 1, 3000, "cuda", hkv=2)
    for _ in range(3):
        assert torch.equal(kv4.decode_attention(q, cache, n, workspace=ws), want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(kv4.decode_attention(q, cache, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ------------------------------------------------------------------ index lists and proxies
def _list_case(g, BQ, BH, Lmax, n_sel, n_exp, NB, per_qhead):
    cache = _records(g, BH, Lmax)
    q = _rows(g, BQ, D)
    sel = torch.randint(-1, Lmax, (BQ, n_sel), generator=g).int()
    exp = torch.randint(-1, Lmax, (BQ, n_exp), generator=g).int()
    if n_exp:
        exp[:, -1] = Lmax                 # outside: padding
    rows = BQ if per_qhead else BH
    kbar, vbar = _rows(g, rows, NB, D), _rows(g, rows, NB, D)
    log_n = torch.rand(BQ, NB, generator=g) * 6
    if NB:
        log_n[:, ::5] = -math.inf
    return q, cache, sel, exp, kbar, vbar, log_n


def _list_want(x, NB, scale=D ** -0.5):
    q, cache, sel, exp, kbar, vbar, log_n = x
    out, slack = torch.zeros(q.shape[0], D, dtype=torch.float64), torch.zeros(q.shape[0], D, dtype=torch.float64)
    G = q.shape[0] // cache.shape[0]
    for r in range(q.shape[0]):
        i = torch.cat([sel[r], exp[r]]).long()
        i = i[(i >= 0) & (i < cache.shape[1])]
        pr = r if kbar.shape[0] == q.shape[0] else r // G
        out[r], slack[r] = P.attend(q[r], cache[r // G, i], scale, kbar[pr, :NB], vbar[pr, :NB], log_n[r, :NB])
    return out, slack


@pytest.mark.parametrize("BQ,BH,Lmax,n_sel,n_exp,NB,per_qhead", [
    (32, 8, 500, 15, 216, 64, True), (6, 2, 40, 1, 0, 0, True), (8, 8, 33, 0, 31, 3, False), (7, 1, 900, 33, 1335, 192, True),
    (4, 2, 300, 9, 23, 65, False), (600, 8, 64, 3, 30, 16, True), (2, 1, 1, 2, 3, 1, True), (16, 1, 200, 70, 64, 10, False)])
def test_flash_attention_lists(BQ, BH, Lmax, n_sel, n_exp, NB, per_qhead):
    x = _list_case(_gen(BQ + n_exp), BQ, BH, Lmax, n_sel, n_exp, NB, per_qhead)
    for out_dtype in (BF, torch.float32):
        got = kv4.flash_attention(*(t.cuda() for t in x), out_dtype=out_dtype)
        P.check(got, *_list_want(x, NB))
    if NB > 1:
        P.check(kv4.flash_attention(*(t.cuda() for t in x), nb=NB - 1), *_list_want(x, NB - 1))
        P.check(kv4.flash_attention(*(t.cuda() for t in x), nb=0, sm_scale=0.3), *_list_want(x, 0, 0.3))


def test_flash_attention_empty_rows_and_repeats():
    """Rows with nothing to attend give zeros; an index listed twice counts twice; proxies alone."""
    x = list(_list_case(_gen(31), 8, 2, 50, 12, 20, 9, True))
    q, cache, sel, exp, kbar, vbar, log_n = x
    sel[0], exp[0], log_n[0] = -1, -1, -math.inf
    sel[1], exp[1], log_n[1] = 7, 7, -math.inf
    sel[2], exp[2] = -1, 50
    sel[3], exp[3], log_n[3] = -1, -1, -math.inf
    exp[3, 19] = 4
    got = kv4.flash_attention(*(t.cuda() for t in x))
    assert not got[0].any()
    P.check(got, *_list_want(x, 9))
    none = torch.zeros(8, 0, dtype=torch.int32, device="cuda")
    assert not kv4.flash_attention(q.cuda(), cache.cuda(), none, none, None, None, None).any()


def test_flash_attention_strided_cache_and_out():
    g = _gen(32)
    x = list(_list_case(g, 8, 2, 60, 5, 40, 7, True))
    big = torch.full((2, 90, REC), 255, dtype=torch.uint8)
    big[:, :60] = x[1]
    wide_k, wide_v = torch.zeros(8, 7, 2 * D, dtype=BF), torch.zeros(8, 7, 2 * D, dtype=BF)
    wide_k[..., :D], wide_v[..., :D] = x[4], x[5]
    buf = torch.full((8, 2 * D), 5.0, device="cuda")
    got = kv4.flash_attention(x[0].cuda(), big.cuda()[:, :60], x[2].cuda(), x[3].cuda(), wide_k.cuda()[..., :D],
                              wide_v.cuda()[..., :D], x[6].cuda(), out=buf[:, :D])
    P.check(got, *_list_want(x, 7))
    assert (buf[:, D:] == 5).all()


def test_lists_of_everything_match_dense():
    """A list of all positions is the dense attention: the two kernels agree within their roundings."""
    g = _gen(33)
    n = 210
    cache = _records(g, 2, n).cuda()
    q = _rows(g, 8, D).cuda()
    every = torch.arange(n, dtype=torch.int32, device="cuda").expand(8, n).contiguous()
    none = torch.zeros(8, 0, dtype=torch.int32, device="cuda")
    a = kv4.flash_attention(q, cache, none, every, None, None, None, out_dtype=torch.float32)
    b = kv4.decode_attention(q.view(1, 8, 1, D), cache.view(1, 2, n, REC), torch.tensor([n], device="cuda"),
                             out_dtype=torch.float32).view(8, D)
    x = (q.cpu(), cache.cpu(), none.cpu(), every.cpu(), torch.zeros(8, 0, D), torch.zeros(8, 0, D), torch.zeros(8, 0))
    want, slack = _list_want(x, 0)
    P.check(a, want, slack)
    P.check(b, want, slack)


# ------------------------------------------------------------------ a run of them, captured and replayed
def test_decode_steps_in_a_graph():
    """Prompt rows enter the cache, then a captured step (rotate, write, attend; two layers that share a
    workspace) is replayed as its position advances; every step equals the eager calls on a second cache."""
    g = _gen(41)
    B, HQ, HKV, T0, steps, Lmax = 2, 8, 2, 37, 6, 64
    cos, sin = (t.cuda() for t in P.table(Lmax, 128))
    zero = torch.zeros(1, dtype=torch.int64, device="cuda")
    k0, v0 = _rows(g, B, HKV, T0, D).cuda(), _rows(g, B, HKV, T0, D).cuda()
    caches = [[kv4.new_cache(B, Lmax, "cuda", hkv=HKV) for _ in range(2)] for _ in range(2)]
    for two in caches:
        for c in two:
            kv4.append(c, k0, v0, zero)
    x = torch.zeros(B, HQ + 2 * HKV, 1, D, dtype=BF, device="cuda")
    pos = torch.full((1,), T0, dtype=torch.int64, device="cuda")  # the warm-up's record is written again by step 0
    ws = kv4.attention_workspace(B, HQ, 1, Lmax, "cuda", hkv=HKV)

    def step(two, at, x, ws):
        outs = []
        for c in two:
            q = kv4.rope_append(c, x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:], cos, sin, at)
            outs.append(kv4.decode_attention(q, c, at, offset=1, workspace=ws))
        return outs

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(caches[0], pos, x, ws)
    torch.cuda.current_stream().wait_stream(s)
    pos.sub_(1)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pos.add_(1)
        outs = step(caches[0], pos, x, ws)
    with torch.cuda.graph(other):  # a second graph of the same sizes, its workspaces its own
        again = step(caches[0], pos, x, None)
    for i in range(steps):
        x.copy_(_rows(g, B, HQ + 2 * HKV, 1, D))
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert int(pos) == T0 + i
        want = step(caches[1], torch.tensor([T0 + i], device="cuda"), x, None)
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert all(torch.equal(a, b) for a, b in zip(again, want))
        assert torch.equal(caches[0][1], caches[1][1])
    rec = caches[1][0].cpu()
    q = rotary.qk_norm_rope(x[:, :HQ], x[:, HQ:HQ + HKV], cos, sin, pos)[0].cpu()
    P.check(outs[0], *_dense_want(q, rec, [T0 + steps] * B, D ** -0.5))


def test_zero_sized_calls():
    z = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = kv4.new_cache(2, 8, "cuda", hkv=2)
    e = torch.zeros(2, 4, 0, D, dtype=BF, device="cuda")
    cos, sin = (t.cuda() for t in P.table(8, 128))
    assert rotary.qk_norm_rope(e, e[:, :2], cos, sin, z)[0].shape == e.shape
    kv4.append(cache, e[:, :2], e[:, :2], z)
    assert kv4.unpack(cache, z, 0)[0].shape == (2, 2, 0, D)
    assert kv4.decode_attention(e, cache, z).shape == e.shape
    q = torch.ones(2, 4, 1, D, dtype=BF, device="cuda")
    assert not kv4.decode_attention(q, cache[:, :, :0], z + 5).any()
    assert not kv4.decode_attention(q, cache, z).any()


def test_dense_long_rows_keep_their_precision():
    """300 heads read one 131072-token row each (the same records, by an expanded cache), so a CTA sums a whole row.
    The fp16 roundings of the weights are independent, each at most 2^-11 of weight * scale * code: their sum has a
    root mean square of at most 2^-11 / sqrt(3) of the root of the summed squares.  Twice 2^-11 is over three times
    that; a bias that grows with the number of tokens is far above it."""
    g = torch.Generator(device="cuda")
    g.manual_seed(51)
    n, H = 131072, 300
    k = torch.randn(n, D, generator=g, device="cuda") + 1.5 * torch.randn(D, generator=g, device="cuda")
    v = torch.randn(n, D, generator=g, device="cuda")
    cache = kv4.new_cache(1, n, "cuda", hkv=1)
    kv4.append(cache, k.to(BF).view(1, 1, n, D), v.to(BF).view(1, 1, n, D), torch.zeros(1, dtype=torch.int32, device="cuda"))
    q = torch.randn(1, H, 1, D, generator=g, device="cuda").to(BF)
    got = kv4.decode_attention(q, cache.expand(1, H, n, REC), torch.tensor([n], device="cuda"), out_dtype=torch.float32)
    K, V = P.values(cache[0, 0], 0), P.values(cache[0, 0], 1)
    code, s, _ = P.parts(cache[0, 0], 1)
    for h in range(0, H, 37):
        w = torch.softmax(K @ q[0, h, 0].double() * D ** -0.5, 0)
        err = (got[0, h, 0].double() - w @ V).norm()
        assert err <= 2 * 2.0 ** -11 * ((w[:, None] * s * code).square().sum().sqrt())


@pytest.mark.parametrize("B,HQ,HKV,T,top", [(100, 8, 8, 1, 60), (90, 64, 8, 2, 40), (700, 1, 1, 1, 300), (75, 40, 8, 1, 33)])
def test_dense_many_short_rows(B, HQ, HKV, T, top):
    """Enough short rows that single warps take them; some requests are empty."""
    g = _gen(B + HQ)
    lens = torch.randint(0, top + 1, (B,), generator=g)
    cache = _records(g, B, HKV, top)
    for b in range(B):
        cache[b, :, int(lens[b]):] = 255
    q = _rows(g, B, HQ, T, D)
    for out_dtype in (BF, torch.float32):
        got = kv4.decode_attention(q.cuda(), cache.cuda(), lens.cuda(), out_dtype=out_dtype).cpu()
        for i in range(0, B * HQ * T, 53):
            b, h, t = i // (HQ * T), i // T % HQ, i % T
            m = max(0, int(lens[b]) - T + 1 + t)
            P.check(got[b, h, t], *P.attend(q[b, h, t], cache[b, h // (HQ // HKV), :m], D ** -0.5))


def test_dense_calls_of_any_size_share_a_workspace():
    """Sizes large, small, ragged and large again, through the kept workspace and through one of the caller's."""
    g = _gen(61)
    ws = kv4.attention_workspace(40, 32, 2, 700, "cuda")
    for B, HQ, HKV, T, top in ((40, 32, 8, 2, 700), (1, 4, 2, 1, 2500), (7, 16, 8, 1, 90), (40, 32, 8, 2, 650), (2, 8, 8, 1, 1300)):
        lens = torch.randint(1, top + 1, (B,), generator=g)
        cache, q = _records(g, B, HKV, top), _rows(g, B, HQ, T, D)
        a = kv4.decode_attention(q.cuda(), cache.cuda(), lens.cuda(), workspace=ws)
        b = kv4.decode_attention(q.cuda(), cache.cuda(), lens.cuda())
        assert torch.equal(a, b)
        for i in range(0, B * HQ * T, 1 + B * HQ * T // 9):
            bb, h, t = i // (HQ * T), i // T % HQ, i % T
            m = max(0, int(lens[bb]) - T + 1 + t)
            P.check(a.cpu()[bb, h, t], *P.attend(q[bb, h, t], cache[bb, h // (HQ // HKV), :m], D ** -0.5))


def test_append_long_odd_heads():
    """A prompt long enough that a warp takes several heads of a token, an odd number of them."""
    g = _gen(62)
    B, T, hkv = 2, 2500, 7
    x = _rows(g, B, T, 2 * hkv, D).transpose(1, 2)
    k, v = x[:, :hkv], x[:, hkv:]
    cache = torch.randint(0, 256, (B, hkv, T + 9, REC), generator=g).to(torch.uint8)
    want = cache.clone()
    want[:, :, 4:4 + T] = P.pack(k, v)
    dev, y = cache.cuda(), x.cuda()
    kv4.append(dev, y[:, :hkv], y[:, hkv:], torch.tensor([5], device="cuda"), offset=-1)
    assert torch.equal(dev.cpu(), want)


@pytest.mark.parametrize("R", [128, 80])
def test_rope_append_long_odd_heads(R):
    """As above for the rotation: one launch equals rotation and append, and both the definition."""
    g = _gen(63)
    B, T, HQ, HKV = 1, 1700, 9, 3
    cos, sin = P.table(T + 3, R)
    x = _rows(g, B, T, HQ + 2 * HKV, D)
    y = x.cuda().transpose(1, 2)
    q, k, v = y[:, :HQ], y[:, HQ:HQ + HKV], y[:, HQ + HKV:]
    w = torch.randn(D, generator=g) + 1
    start = torch.tensor([3], dtype=torch.int32, device="cuda")
    one, two = kv4.new_cache(B, T + 3, "cuda", hkv=HKV), kv4.new_cache(B, T + 3, "cuda", hkv=HKV)
    args = dict(q_weight=w.cuda(), k_weight=w.cuda())
    q1 = kv4.rope_append(one, q, k, v, cos.cuda(), sin.cuda(), start, **args)
    q2, k2 = rotary.qk_norm_rope(q, k, cos.cuda(), sin.cuda(), start, **args)
    kv4.append(two, k2, v, start)
    assert torch.equal(q1, q2) and torch.equal(one, two)
    for got, h0, h1 in ((q2, 0, HQ), (k2, HQ, HQ + HKV)):
        P.check(got, *P.rope(x.transpose(1, 2)[:, h0:h1], cos, sin, [3], [T], w))


@pytest.mark.parametrize("B,HKV,lens", [
    (310, 1, [700, 0, 3, 64, 1, 33, 250, 90, 5, 12]),   # more rows than CTAs, too uneven for a warp each: shares of a line
    (16, 8, [5000, 1, 0, 33, 900, 64, 2, 400]),         # rows with CTAs to spare, too uneven to have their own
    (40, 8, [1100, 1300, 1200])])                       # even ones on the line
def test_dense_rows_that_share_ctas(B, HKV, lens):
    g = _gen(64 + B)
    lens = [lens[b % len(lens)] if b % 7 else lens[0] for b in range(B)]
    cache = _records(g, B, HKV, max(lens))
    q = _rows(g, B, HKV, 1, D)
    got = kv4.decode_attention(q.cuda(), cache.cuda(), torch.tensor(lens, device="cuda"), out_dtype=torch.float32)
    step = 1 if HKV == 1 else 5
    want, slack = _dense_want(q[:, ::step], cache[:, ::step], lens, D ** -0.5)
    P.check(got[:, ::step], want, slack)


@pytest.mark.parametrize("BQ,n_exp", [(30, 1300), (60, 1300), (8, 2000), (100, 700)])
def test_lists_of_few_rows(BQ, n_exp):
    """Rows that clusters of 4, 2, 8 and no cluster share."""
    x = _list_case(_gen(BQ + n_exp), BQ, 2, 900, 5, n_exp, 7, True)
    P.check(kv4.flash_attention(*(t.cuda() for t in x), out_dtype=torch.float32), *_list_want(x, 7))


@pytest.mark.parametrize("B,HQ,HKV,T,lens", [
    (3, 4, 2, 2, [1, 33, 700]), (2, 2, 2, 3, [2, 65]), (1, 8, 2, 1, [5]), (4, 3, 3, 4, [4, 3, 0, 40]),
    (600, 1, 1, 4, [50, 3, 0, 64, 33, 1, 2, 17, 96])])
def test_dense_few_columns_of_several_tokens(B, HQ, HKV, T, lens):
    """At most four columns a KV head, from heads and query tokens; the last with a warp to a row."""
    g = _gen(65 + B)
    lens = [lens[b % len(lens)] for b in range(B)]
    cache = _records(g, B, HKV, max(lens))
    for b, n in enumerate(lens):
        cache[b, :, n:] = 255
    q = _rows(g, B, HQ, T, D)
    got = kv4.decode_attention(q.cuda(), cache.cuda(), torch.tensor(lens, device="cuda"), out_dtype=torch.float32)
    P.check(got, *_dense_want(q, cache, lens, D ** -0.5))


def test_prompt_write_read_and_lists_in_a_graph():
    """Rotation, cache write, read-back and list attention captured before any of them ran eagerly on these tensors, and
    replayed with new inputs and positions, twice over one graph's outputs."""
    g = _gen(66)
    B, HQ, HKV, T, Lmax = 2, 8, 2, 21, 64
    cos, sin = (t.cuda() for t in P.table(Lmax, 128))
    x = torch.zeros(B, T, HQ + 2 * HKV, D, dtype=BF, device="cuda")
    start = torch.zeros(B, dtype=torch.int32, device="cuda")
    sel = torch.full((B * HQ, 5), -1, dtype=torch.int32, device="cuda")
    exp = torch.full((B * HQ, 40), -1, dtype=torch.int32, device="cuda")
    kb, vb, ln = (torch.zeros(B * HQ, 6, D, dtype=BF, device="cuda"), torch.zeros(B * HQ, 6, D, dtype=BF, device="cuda"),
                  torch.zeros(B * HQ, 6, device="cuda"))
    cache = kv4.new_cache(B, Lmax, "cuda", hkv=HKV)

    def run(cache):
        y = x.transpose(1, 2)
        q, k = rotary.qk_norm_rope(y[:, :HQ], y[:, HQ:HQ + HKV], cos, sin, start)
        kv4.append(cache, k, y[:, HQ + HKV:], start)
        k2, v2 = kv4.unpack(cache, start, T)
        o = kv4.flash_attention(q[:, :, -1].reshape(B * HQ, D), cache.view(B * HKV, Lmax, REC), sel, exp, kb, vb, ln)
        return q, k2, v2, o

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(cache)
    other = kv4.new_cache(B, Lmax, "cuda", hkv=HKV)
    for i in range(3):
        x.copy_(_rows(g, B, T, HQ + 2 * HKV, D))
        start.copy_(torch.tensor([3 * i, 40 - i]))
        sel.copy_(torch.randint(-1, Lmax, sel.shape, generator=g))
        exp.copy_(torch.randint(-1, Lmax, exp.shape, generator=g))
        kb.copy_(_rows(g, B * HQ, 6, D))
        vb.copy_(_rows(g, B * HQ, 6, D))
        graph.replay()
        torch.cuda.synchronize()
        want = run(other)
        assert torch.equal(cache, other) and all(torch.equal(a, b) for a, b in zip(outs, want))
