"""Attention over the 4-bit cache where rows differ by many powers of two: a record whose V scale is far above the
others' and whose weight makes up for it, against the definition in 64 bits (kv4_plain.py derives the tolerances)."""
import math

import pytest
import torch

import kv4_plain as P
from openattention_b200 import kv4

pytestmark = pytest.mark.gpu
D, REC = 128, 144
BF = torch.bfloat16


def _far_apart(seed, heads, n, power, early):
    """q (heads, 128) and records (n, 144).  The record at `at` has V values 2^power times the others'.

    early: it is the first, its logit like its neighbours', and the second half of the tokens stand 60 (nats) above it:
    by then its weight is 2^-86.  Else its own logit lies about 40 below the others'."""
    g = torch.Generator().manual_seed(seed)
    u = torch.randint(0, 2, (D,), generator=g) * 2.0 - 1
    q = u + torch.randn(heads, D, generator=g) * 0.25
    k, v = torch.randn(n, D, generator=g), torch.randn(n, D, generator=g)
    at = 0 if early else n // 3
    if early:
        k[n // 2:] += u * 60 / (D * D ** -0.5)
    else:
        k[at] = -u * 40 / (D * D ** -0.5) + torch.randn(D, generator=g) * 0.1
    v[at] *= 2.0 ** power
    return q.to(BF), P.pack(k.to(BF), v.to(BF))


FAR = [(26, False), (40, False), (26, True), (70, True)]


@pytest.mark.parametrize("power,early", FAR)
@pytest.mark.parametrize("B,HKV,G,T,n", [
    (1, 1, 4, 1, 4096),      # a tile or two a warp, many parts
    (16, 8, 2, 1, 4000),     # several tiles a warp
    (16, 8, 8, 1, 4000), (16, 8, 3, 2, 4000),  # eight columns
    (100, 4, 4, 1, 330), (100, 4, 7, 1, 330)])  # a warp a row
def test_dense_values_far_apart(B, HKV, G, T, n, power, early):
    q, rec = _far_apart(71 + G, HKV * G * T, n, power, early)
    q = q.view(1, HKV * G, T, D)
    got = kv4.decode_attention(q.cuda().expand(B, -1, -1, -1), rec.cuda().expand(B, HKV, n, REC),
                               torch.tensor([n], device="cuda"), out_dtype=torch.float32).cpu()
    assert torch.equal(got, got[:1].expand_as(got))
    for h in range(0, HKV * G, 1 + HKV * G // 6):
        for t in range(T):
            P.check(got[0, h, t], *P.attend(q[0, h, t], rec[:n - T + 1 + t], D ** -0.5), f"head {h}, token {t}")


@pytest.mark.parametrize("power,early", FAR)
@pytest.mark.parametrize("rows,n,NB", [(2, 2000, 0), (40, 1300, 7), (200, 700, 9), (1100, 231, 64)])
def test_lists_values_far_apart(rows, n, NB, power, early):
    q, rec = _far_apart(72 + rows, rows, n, power, early)
    g = torch.Generator().manual_seed(73)
    kbar, vbar = torch.randn(rows, NB, D, generator=g).to(BF), torch.randn(rows, NB, D, generator=g).to(BF)
    # with `early`, proxies stand where the late tokens do
    log_n = torch.rand(rows, NB, generator=g) * 3 + (60 if early else 0)
    idx = torch.arange(n, dtype=torch.int32).expand(rows, n).contiguous()
    got = kv4.flash_attention(q.cuda(), rec.cuda()[None], idx[:, :5].contiguous().cuda(), idx[:, 5:].contiguous().cuda(),
                              kbar.cuda(), vbar.cuda(), log_n.cuda(), out_dtype=torch.float32).cpu()
    for r in range(0, rows, 1 + rows // 9):
        P.check(got[r], *P.attend(q[r], rec, D ** -0.5, kbar[r], vbar[r], log_n[r]), f"row {r}")


@pytest.mark.parametrize("vs,ps", [(1.0, 1e25), (1.0, 1e30), (1e30, 1e30), (1.0, 1e35), (1e30, 1.0), (1e-30, 1.0), (1.0, 1e-30),
                                   (1e-30, 1e-30)])
@pytest.mark.parametrize("n,NB", [(300, 20), (0, 9), (70, 3)])
def test_lists_large_and_small_value_rows(n, NB, vs, ps):
    """Values of the records and of the proxies far from 1, and from each other."""
    g = torch.Generator().manual_seed(74)
    rows = 6
    rec = P.pack(torch.randn(400, D, generator=g).to(BF), (torch.randn(400, D, generator=g) * vs).to(BF))
    q, kbar = torch.randn(rows, D, generator=g).to(BF), torch.randn(rows, NB, D, generator=g).to(BF)
    vbar = (torch.randn(rows, NB, D, generator=g) * ps).to(BF)
    log_n = torch.rand(rows, NB, generator=g) * 3
    log_n[:2] = -math.inf                # rows without proxies
    idx = torch.arange(n, dtype=torch.int32).expand(rows, n).contiguous()
    none = torch.zeros(rows, 0, dtype=torch.int32)
    for out_dtype in (BF, torch.float32):
        got = kv4.flash_attention(q.cuda(), rec.cuda()[None], none.cuda(), idx.cuda(), kbar.cuda(), vbar.cuda(), log_n.cuda(),
                                  out_dtype=out_dtype).cpu()
        for r in range(rows):
            P.check(got[r], *P.attend(q[r], rec[:n], D ** -0.5, kbar[r], vbar[r], log_n[r]), f"row {r}")


@pytest.mark.parametrize("G", [2, 8])
@pytest.mark.parametrize("half,power", [(0, -30), (1, -26)])
def test_query_elements_far_apart(G, half, power):
    """A query element of 1 meets codes of 0 only; what decides are the others, 2^-30 of it (dims 0..63) or 2^-26 (64..127),
    which the fp16 operand still holds in full."""
    g = torch.Generator().manual_seed(75)
    n, H = 500, 4
    q = torch.zeros(1, H * G, 1, D)
    q[..., 64 * half:64 * half + 64] = (1 + torch.rand(1, H * G, 1, 64, generator=g)) * 2.0 ** power * (
        torch.randint(0, 2, (1, H * G, 1, 64), generator=g) * 2 - 1)
    q[..., 0] = 1.0
    k = torch.zeros(1, H, n, D)
    k[..., 64 * half:64 * half + 64] = torch.rand(1, H, n, 64, generator=g) * 2
    k[..., 64 * half + 63] = 0.0          # the group's minimum, so its offset, is 0
    k[..., 0] = 0.0
    q, cache = q.to(BF), P.pack(k.to(BF), torch.randn(1, H, n, D, generator=g).to(BF))
    scale = 0.25 * 2.0 ** -power
    got = kv4.decode_attention(q.cuda(), cache.cuda(), torch.tensor([n], device="cuda"), sm_scale=scale, out_dtype=torch.float32)
    for h in range(H * G):
        P.check(got[0, h, 0], *P.attend(q[0, h, 0], cache[0, h // G], scale), f"head {h}")


@pytest.mark.parametrize("scale", [D ** -0.5, 3.7, -0.01])
@pytest.mark.parametrize("G,T", [(1, 1), (4, 1), (8, 1), (3, 2)])
def test_one_token_gives_its_values(G, T, scale):
    """A softmax over one token, or over copies of one, is the token's values: the weight is 1 and its product with a bf16
    scale holds in fp16, so only fp32 roundings remain (of scale * code + offset, in up to four steps, and the division)."""
    g = torch.Generator().manual_seed(76)
    B, H, n = 3, 4, 9
    rec = P.pack(*(torch.randn(B, H, 1, D, generator=g).to(BF) for _ in range(2)))
    q = torch.randn(B, H * G, T, D, generator=g).to(BF)
    code, s, z = (t.repeat_interleave(G, 1) for t in P.parts(rec, 1))  # (B, H * G, 1, 128)
    want, slack = s * code + z, 8 * 2.0 ** -24 * (15 * s + z.abs())
    for m in (1, n):
        lens = torch.full((B,), m + T - 1, dtype=torch.int32, device="cuda")
        got = kv4.decode_attention(q.cuda(), rec.cuda().expand(B, H, 1, REC).repeat(1, 1, n + T, 1), lens, sm_scale=scale,
                                   out_dtype=torch.float32)
        P.check(got[:, :, :1], want, slack, f"{m} tokens")
        i = torch.zeros(B * H * G, m, dtype=torch.int32, device="cuda")
        got = kv4.flash_attention(q[:, :, 0].reshape(-1, D).cuda(), rec.view(B * H, 1, REC).cuda(), i[:, :0], i, None, None, None,
                                  sm_scale=scale, out_dtype=torch.float32)
        P.check(got.view(B, H * G, 1, D), want, slack, f"list of {m}")
