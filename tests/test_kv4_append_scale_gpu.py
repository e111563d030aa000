"""The cache write where the scale is rounded furthest: down by nearly 2^-8 of it, so that the largest quotient stands
furthest above 15, or up, so that it falls furthest below."""
import pytest
import torch

import kv4_plain as P
from openattention_b200 import kv4

pytestmark = pytest.mark.gpu
D, BF = 128, torch.bfloat16


@pytest.mark.parametrize("hkv,T", [(1, 1), (3, 40)])
@pytest.mark.parametrize("power", [0, -100, 100, 7])
@pytest.mark.parametrize("low,scale,largest", [
    (-0.05859375, 1.0, 15.05859375),             # (max - min) / 15 = 1 + 2^-8, half a step above 1: to even, 1
    (-0.058349609375, 1.0, 15.058349609375),     # just under it
    (-0.06201171875, 1.0078125, 14.945),         # and just above it
])
def test_scale_rounded_furthest(hkv, T, power, low, scale, largest):
    g = torch.Generator().manual_seed(91)
    x = torch.rand(2, 1, hkv, T, D, generator=g) * 15
    x[..., 0::64] = 15.0
    x[..., 63::64] = low
    x = (x * 2.0 ** power).to(BF)
    code, s, z = P.quantise(x)
    assert (s == scale * 2.0 ** power).all() and code.max() == 15 and (code[..., 0::64] == 15).all()
    quotient = (15 * 2.0 ** power - z.double()) / s.double()
    assert ((quotient - largest).abs() < 1e-3).all()
    cache = kv4.new_cache(1, T, "cuda", hkv=hkv)
    kv4.append(cache, x[0].cuda(), x[1].cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert torch.equal(cache.cpu(), P.pack(x[0], x[1]))
    cos, sin = torch.ones(T, D, device="cuda"), torch.zeros(T, D, device="cuda")  # no rotation: k as it is
    other = kv4.new_cache(1, T, "cuda", hkv=hkv)
    kv4.rope_append(other, x[0].cuda(), x[0].cuda(), x[1].cuda(), cos, sin, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert torch.equal(other, cache)
