"""Rows rotated where they stand: the same bits as into other memory, at sizes where a warp takes several rows of a token,
an odd number of them (its last loads then read a row again that it has already written)."""
import pytest
import torch

import kv4_plain as P
from openattention_b200 import kv4, rotary

pytestmark = pytest.mark.gpu
D, BF = 128, torch.bfloat16


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("B,T,HQ,HKV,R,norm", [(1, 1, 32, 8, 128, False), (2, 3000, 9, 3, 128, True), (1, 5000, 33, 7, 128, False),
                                               (1, 4000, 15, 1, 48, True)])
def test_in_place_is_the_same_bits(B, T, HQ, HKV, R, norm, dtype):
    g = torch.Generator().manual_seed(81)
    cos, sin = (t.cuda() for t in P.table(T + 4, R))
    x = torch.randn(B, T, HQ + 2 * HKV, D, generator=g).to(dtype).cuda()
    w = dict(q_weight=(torch.randn(D, generator=g) + 1).cuda(), k_weight=(torch.randn(D, generator=g) + 1).cuda()) if norm else {}
    start = torch.tensor([3], device="cuda")
    lens = torch.tensor([T - b for b in range(B)], device="cuda")

    def parts(x):
        y = x.transpose(1, 2)
        return y[:, :HQ], y[:, HQ:HQ + HKV], y[:, HQ + HKV:]

    y = x.clone()
    (q, k, v), (q2, k2, v2) = parts(x), parts(y)
    want = [t.clone() for t in (q, k)]
    rotary.qk_norm_rope(q, k, cos, sin, start, lens=lens, q_out=want[0], k_out=want[1], **w)
    rotary.qk_norm_rope(q2, k2, cos, sin, start, lens=lens, q_out=q2, k_out=k2, **w)
    assert torch.equal(q2, want[0]) and torch.equal(k2, want[1]) and torch.equal(v2, v)
    if dtype is BF:
        y = x.clone()
        q2, k2, v2 = parts(y)
        one, two = kv4.new_cache(B, T + 4, "cuda", hkv=HKV), kv4.new_cache(B, T + 4, "cuda", hkv=HKV)
        kv4.rope_append(one, q, k, v, cos, sin, start, lens=lens, **w)
        kv4.rope_append(two, q2, k2, v2, cos, sin, start, lens=lens, q_out=q2, **w)
        assert torch.equal(one, two) and torch.equal(q2, want[0]) and torch.equal(k2, k) and torch.equal(v2, v)
