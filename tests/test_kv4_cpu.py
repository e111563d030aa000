"""What the 4-bit cache operators and the rotation refuse, before any launch; and the definitions the GPU tests
compare with, checked on the CPU."""
import ctypes

import pytest
import torch

import kv4_plain as P
from openattention_b200 import _lib, kv4, rotary

D, REC, BF = 128, 144, torch.bfloat16


def test_wrappers_refuse_host_tensors():
    q, k = torch.zeros(1, 4, 2, D, dtype=BF), torch.zeros(1, 2, 2, D, dtype=BF)
    cos, sin = P.table(8, 128)
    z = torch.zeros(1, dtype=torch.int32)
    cache = torch.zeros(1, 2, 8, REC, dtype=torch.uint8)
    idx = torch.zeros(4, 3, dtype=torch.int32)
    for call in (lambda: rotary.qk_norm_rope(q, k, cos, sin, z), lambda: kv4.append(cache, k, k, z),
                 lambda: kv4.rope_append(cache, q, k, k, cos, sin, z), lambda: kv4.unpack(cache, z, 2),
                 lambda: kv4.decode_attention(q, cache, z),
                 lambda: kv4.flash_attention(q[0, :, 0], cache[0], idx, idx, None, None, None)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


class _Fake(torch.Tensor):
    """A host tensor that says it is on a GPU: the checks behind the device's own are reached without one."""
    is_cuda = True


def _fake(t):
    return t.as_subclass(_Fake)


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(1, 4, 2, D, dtype=torch.float16)), "q must be torch.bfloat16"),
    (dict(q=torch.zeros(4, 2, D, dtype=BF)), "q must be"),
    (dict(q=torch.zeros(1, 4, 2, 64, dtype=BF)), "q must be"),
    (dict(q=torch.zeros(1, 4, D, 2, dtype=BF).transpose(2, 3)), "contiguous last dim"),
    (dict(k=torch.zeros(1, 2, 3, D, dtype=BF)), "k must be"),
    (dict(k=torch.zeros(1, 2, 2, D)), "k must be torch.bfloat16"),
    (dict(start=torch.zeros(3, dtype=torch.int32)), "start must be"),
    (dict(start=torch.zeros(1)), "start must be"),
    (dict(start=0), "start must be"),
    (dict(lens=torch.zeros(1, 1, dtype=torch.int32)), "lens must be"),
    (dict(cos=torch.zeros(8, 64)), "must be a contiguous fp32"),
    (dict(q_weight=torch.zeros(64)), "norm weights"),
    (dict(q_weight=torch.zeros(D), k_weight=torch.zeros(D, dtype=BF)), "norm weights"),
    (dict(q_out=torch.zeros(1, 4, 2, D)), "q_out must be torch.bfloat16"),
    (dict(q_out=torch.zeros(1, 1, 2, D, dtype=BF).expand(1, 4, 2, D)), "expanded"),
])
def test_rope_refusals(change, match):
    a = dict(q=torch.zeros(1, 4, 2, D, dtype=BF), k=torch.zeros(1, 2, 2, D, dtype=BF), start=torch.zeros(1, dtype=torch.int32))
    a["cos"], a["sin"] = P.table(8, 128)
    a.update(change)
    with pytest.raises(RuntimeError, match=match):
        rotary.qk_norm_rope(**{n: _fake(t) if isinstance(t, torch.Tensor) else t for n, t in a.items()})


def test_gradients_are_refused():
    q = _fake(torch.zeros(1, 4, 2, D, dtype=BF)).requires_grad_()
    k = _fake(torch.zeros(1, 2, 2, D, dtype=BF))
    cos, sin = P.table(8, 128)
    with pytest.raises(RuntimeError, match="no backward pass"):
        rotary.qk_norm_rope(q, k, cos, sin, torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("cache,match", [
    (torch.zeros(1, 2, 8, REC), "uint8"), (torch.zeros(1, 2, 8, 160, dtype=torch.uint8)[..., :REC], "contiguous records"),
    (torch.zeros(2, 8, REC, dtype=torch.uint8), "cache must be"), (torch.zeros(1, 2, 8, 128, dtype=torch.uint8), "cache must be"),
    (torch.zeros(1, 1, 8, REC, dtype=torch.uint8).expand(1, 2, 8, REC), "expanded")])
def test_append_refuses_caches(cache, match):
    k = _fake(torch.zeros(1, 2, 2, D, dtype=BF))
    with pytest.raises(RuntimeError, match=match):
        kv4.append(_fake(cache), k, k, _fake(torch.zeros(1, dtype=torch.int32)))


@pytest.mark.parametrize("change,match", [
    (dict(cache=torch.zeros(2, 2, 8, REC, dtype=torch.uint8)), "same requests"),
    (dict(cache=torch.zeros(1, 3, 8, REC, dtype=torch.uint8)), "multiple of the KV heads"),
    (dict(n=None), "n must be given"), (dict(n=torch.zeros(2, dtype=torch.int32)), "n must be"),
    (dict(out_dtype=torch.float16), "bf16 or fp32"), (dict(out=torch.zeros(1, 4, 1, D, dtype=BF)), "out must be"),
    (dict(out=torch.zeros(1, 4, 2, D, dtype=BF), out_dtype=torch.float32), "out_dtype"),
    (dict(workspace=torch.zeros(4)), "workspace")])
def test_decode_attention_refusals(change, match):
    a = dict(q=torch.zeros(1, 4, 2, D, dtype=BF), cache=torch.zeros(1, 2, 8, REC, dtype=torch.uint8),
             n=torch.zeros(1, dtype=torch.int32))
    a.update(change)
    with pytest.raises(RuntimeError, match=match):
        kv4.decode_attention(**{n: _fake(t) if isinstance(t, torch.Tensor) else t for n, t in a.items()})


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(4, D)), "q must be"), (dict(cache=torch.zeros(3, 8, REC, dtype=torch.uint8)), "multiple of the cache's"),
    (dict(sel_idx=torch.zeros(4, 2, dtype=torch.int64)), "sel_idx"), (dict(exp_idx=torch.zeros(3, 2, dtype=torch.int32)), "exp_idx"),
    (dict(nb=9), "kbar must be"), (dict(nb=-1), "nb must not"), (dict(vbar=torch.zeros(4, 5, D, dtype=BF)), "vbar"),
    (dict(log_n=torch.zeros(4, 4)), "log_n"), (dict(out=torch.zeros(4, 64)), "out must be")])
def test_flash_attention_refusals(change, match):
    i = torch.zeros(4, 2, dtype=torch.int32)
    a = dict(q=torch.zeros(4, D, dtype=BF), cache=torch.zeros(2, 8, REC, dtype=torch.uint8), sel_idx=i, exp_idx=i,
             kbar=torch.zeros(4, 6, D, dtype=BF), vbar=torch.zeros(4, 6, D, dtype=BF), log_n=torch.zeros(4, 6))
    a.update(change)
    with pytest.raises(RuntimeError, match=match):
        kv4.flash_attention(**{n: _fake(t) if isinstance(t, torch.Tensor) else t for n, t in a.items()})


def _status(name, args, match):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == 1
    assert match in lib.oa_last_error_string(), lib.oa_last_error_string()


def test_c_entries_check_their_arguments():
    """Status 1 and a message, before any device work (the pointers are host addresses)."""
    buf = ctypes.create_string_buffer(4096)
    a = (ctypes.addressof(buf) + 255) // 256 * 256
    f = ctypes.c_float

    def rope(q=a, sb=0, R=128, dtype=0, B=1, HKV=1, start=a, cos=a, w=0):
        return (q, sb, 0, 0, a, 0, 0, 0, a, 0, 0, 0, a, 0, 0, 0, dtype, B, 1, 1, HKV, cos, a, 8, R, start, 0, 0, 0, 0, 0, 0, w, 0,
                1, f(1e-5), 0, 0, None)

    _status("oa_qk_norm_rope", rope(R=24), b"multiple of 16")
    _status("oa_qk_norm_rope", rope(R=144), b"multiple of 16")
    _status("oa_qk_norm_rope", rope(dtype=7), b"dtype")
    _status("oa_qk_norm_rope", rope(q=a + 2), b"16-byte")
    _status("oa_qk_norm_rope", rope(q=0), b"null rows")
    _status("oa_qk_norm_rope", rope(sb=4), b"16-byte")
    _status("oa_qk_norm_rope", rope(HKV=0), b"bad sizes")
    _status("oa_qk_norm_rope", rope(B=-1), b"bad sizes")
    _status("oa_qk_norm_rope", rope(start=0), b"null start")
    _status("oa_qk_norm_rope", rope(cos=a + 4), b"cos/sin")
    _status("oa_qk_norm_rope", rope(w=a + 2), b"weights")

    def append(k=a, cache=a, c_sb=0, HQ=0, cos=0, Lmax=4, start=a):
        return (0, 0, 0, 0, k, 0, 0, 0, a, 0, 0, 0, 0, 0, 0, 0, cache, c_sb, 0, Lmax, 1, 1, HQ, 1, cos, cos, 4, 128, start, 0, 0, 0,
                0, 0, 0, 0, 0, 1, f(0), 0, None)

    _status("oa_kv4_append", append(k=0), b"null rows")
    _status("oa_kv4_append", append(cache=0), b"cache")
    _status("oa_kv4_append", append(cache=a + 8), b"cache")
    _status("oa_kv4_append", append(c_sb=8), b"strides")
    _status("oa_kv4_append", append(Lmax=-1), b"cache length")
    _status("oa_kv4_append", append(HQ=1), b"cos/sin")
    _status("oa_kv4_append", append(HQ=1, cos=a), b"null rows")
    _status("oa_kv4_append", append(start=0), b"null start")

    def unpack(cache=a, out=a, st=128, dtype=0, T=1):
        return (cache, 0, 0, 4, a, 0, 0, 0, 0, 0, 0, out, 0, 0, st, out, 0, 0, 128, dtype, 1, T, 1, 0, 0, None)

    _status("oa_kv4_unpack", unpack(cache=a + 1), b"cache")
    _status("oa_kv4_unpack", unpack(out=0), b"null rows")
    _status("oa_kv4_unpack", unpack(st=6), b"16-byte")
    _status("oa_kv4_unpack", unpack(dtype=3), b"dtype")
    _status("oa_kv4_unpack", unpack(T=-1), b"bad sizes")

    def dense(q=a, cache=a, n=a, HQ=4, HKV=2, out=a, dtype=0, c_sh=144, B=1):
        return (q, 0, 0, 0, cache, 0, c_sh, 64, n, 0, 0, 0, out, 0, 128, 0, dtype, B, HQ, HKV, 1, f(1), 0, 0, None)

    _status("oa_kv4_attention", dense(HQ=5), b"multiple of HKV")
    _status("oa_kv4_attention", dense(HKV=0), b"multiple of HKV")
    _status("oa_kv4_attention", dense(B=-1), b"B, T >= 0")
    _status("oa_kv4_attention", dense(cache=a + 8), b"16 bytes")
    _status("oa_kv4_attention", dense(c_sh=100), b"16 bytes")
    _status("oa_kv4_attention", dense(n=0), b"null q/out/n")
    _status("oa_kv4_attention", dense(q=a + 8), b"16-byte")
    _status("oa_kv4_attention", dense(dtype=2), b"out_dtype")

    def lists(q=a, BQ=4, BH=2, sel=a, NB=0, kbar=0, qs=128, n_exp=0, dtype=1, Lmax=8):
        return (q, qs, a, 8 * REC, Lmax, sel, 1, 0, n_exp, kbar, kbar, 0, 0, 1, kbar, 0, a, 128, dtype, BQ, BH, NB, f(1), None)

    _status("oa_kv4_flash", lists(BQ=3), b"multiple of BH")
    _status("oa_kv4_flash", lists(BH=0), b"multiple of BH")
    _status("oa_kv4_flash", lists(sel=0), b"null index list")
    _status("oa_kv4_flash", lists(n_exp=2), b"null index list")
    _status("oa_kv4_flash", lists(NB=2), b"null kbar")
    _status("oa_kv4_flash", lists(NB=2, kbar=a + 2), b"kbar/vbar")
    _status("oa_kv4_flash", lists(qs=4), b"16-byte")
    _status("oa_kv4_flash", lists(q=0), b"null q")
    _status("oa_kv4_flash", lists(dtype=5), b"out_dtype")
    _status("oa_kv4_flash", lists(Lmax=-1), b"bad list sizes")


def test_plain_record_round_trip():
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(5, D, generator=g).bfloat16(), torch.randn(5, D, generator=g).bfloat16()
    rec = P.pack(k, v)
    assert rec.shape == (5, REC)
    for x, side in ((k, 0), (v, 1)):
        _, s, _ = P.parts(rec, side)
        assert ((P.values(rec, side) - x.double()).abs() <= s / 2 * (1 + 2.0 ** -20)).all()


def test_plain_rope_is_a_rotation():
    """With one angle for both dims of a pair, lengths of pairs are kept."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(1, 2, 3, D, generator=g)
    a = torch.rand(9, 32, generator=g) * 3
    a = torch.cat([a, a], -1)
    y, _ = P.rope(x, a.cos(), a.sin(), [4], [3])
    def size(t):
        return t[..., :32].double() ** 2 + t[..., 32:64].double() ** 2
    assert torch.allclose(size(y), size(x), rtol=1e-6) and torch.equal(y[..., 64:], x[..., 64:].double())
