"""What the 4-bit cache operators and the rotation refuse, before any launch; and the definitions the GPU tests
compare with, checked on the CPU."""
import os
import re

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
    """A host tensor that says it is on a GPU."""
    is_cuda = True


def _fake(t):
    return t.as_subclass(_Fake) if isinstance(t, torch.Tensor) else t


@pytest.fixture
def entry(monkeypatch):
    """Lets wrappers reach the library with host tensors, which every call here must be refused before using: not
    where a GPU could be given their addresses."""
    if torch.cuda.is_available():
        pytest.skip("host addresses are not passed on where there is a GPU")
    for m in (rotary, kv4):
        monkeypatch.setattr(m, "_current_stream", lambda dev: 0)
    monkeypatch.setattr(rotary, "_current_device", lambda: -1)


def _refused(call, base, change, match):
    a = {**base, **change}
    with pytest.raises(RuntimeError, match=match):
        call(**{n: _fake(t) for n, t in a.items()})


def _i(n=1, dtype=torch.int32):
    return torch.zeros(n, dtype=dtype)


def _r(*shape, dtype=BF):
    return torch.zeros(*shape, D, dtype=dtype)


def _c(*shape):
    return torch.zeros(*shape, REC, dtype=torch.uint8)


ROPE = [
    (dict(q=_r(1, 4, 2, dtype=torch.float16)), "q must be torch.bfloat16"),
    (dict(q=_r(4, 2)), "q must be"),
    (dict(q=torch.zeros(1, 4, 2, 64, dtype=BF)), "q must be .* 128"),
    (dict(q=torch.zeros(1, 4, D, D, dtype=BF).transpose(2, 3), k=_r(1, 2, D)), "contiguous last dim"),
    (dict(q=torch.zeros(1 + 4 * 2 * 132, dtype=BF)[1:].view(1, 4, 2, 132)[..., :D]), "16-byte"),
    (dict(k=_r(1, 2, 3)), "k must be"),
    (dict(k=_r(2, 2, 2)), "k must be"),
    (dict(k=_r(1, 2, 2, dtype=torch.float32)), "k must be torch.bfloat16"),
    (dict(start=_i(3)), "start must hold 1"),
    (dict(start=torch.zeros(1)), "start must be"),
    (dict(start=None), "start must be given"),
    (dict(start=0), "start must be"),
    (dict(lens=_i(1).view(1, 1)), "lens must be"),
    (dict(lens=_i(2)), "lens must hold"),
    (dict(cos=torch.zeros(8, 64)), "must be a contiguous fp32"),
    (dict(cos=torch.zeros(8, 24), sin=torch.zeros(8, 24)), "multiple of 16"),
    (dict(cos=torch.zeros(8, 144), sin=torch.zeros(8, 144)), "multiple of 16"),
    (dict(q_weight=torch.zeros(64)), "norm weights"),
    (dict(q_weight=torch.zeros(D), k_weight=torch.zeros(D, dtype=BF)), "norm weights"),
    (dict(q_out=_r(1, 4, 2, dtype=torch.float32)), "q_out must be torch.bfloat16"),
    (dict(q_out=_r(1, 4, 3)), "q_out must be"),
    (dict(q_out=_r(1, 1, 2).expand(1, 4, 2, D)), "expanded"),
    (dict(q_out=_r(5 * 4 * 2).view(-1).as_strided((1, 4, 2, D), (2048, 256, 64, 1))), "overlap"),
    (dict(q=_r(1, 4, 2).requires_grad_()), "no backward pass"),
    (dict(k_weight=torch.zeros(D, requires_grad=True)), "no backward pass"),
    (dict(cos=torch.zeros(8, 128, requires_grad=True)), "no backward pass"),
]


@pytest.mark.parametrize("change,match", ROPE)
def test_rope_refusals(entry, change, match):
    cos, sin = P.table(8, 128)
    _refused(rotary.qk_norm_rope, dict(q=_r(1, 4, 2), k=_r(1, 2, 2), cos=cos, sin=sin, start=_i()), change, match)


@pytest.mark.parametrize("change,match", [
    (dict(cache=torch.zeros(1, 2, 8, REC)), "uint8"),
    (dict(cache=torch.zeros(1, 2, 8, 160, dtype=torch.uint8)[..., :REC]), "contiguous records"),
    (dict(cache=_c(2, 8)), "cache must be"), (dict(cache=torch.zeros(1, 2, 8, 128, dtype=torch.uint8)), "cache must be"),
    (dict(cache=_c(1, 1, 8).expand(1, 2, 8, REC)), "expanded"), (dict(cache=_c(1, 3, 8)), "k must be"),
    (dict(cache=_c(1, 2, 8).as_strided((1, 2, 8, REC), (2 * 8 * REC, 4 * REC, REC, 1))), "share records"),
    (dict(cache=torch.zeros(2 * 8 * REC + 8, dtype=torch.uint8)[8:].view(1, 2, 8, REC)), "16-byte"),
    (dict(v=_r(1, 2, 3)), "v must be"), (dict(start=_i(4)), "start must hold"), (dict(start=None), "start must be given"),
    (dict(lens=torch.zeros(1)), "lens must be")])
def test_append_refusals(entry, change, match):
    _refused(kv4.append, dict(cache=_c(1, 2, 8), k=_r(1, 2, 2), v=_r(1, 2, 2), start=_i()), change, match)


@pytest.mark.parametrize("change,match", [
    (dict(q=_r(1, 4, 3)), "q must be"), (dict(q=_r(1, 4, 2, dtype=torch.float32)), "q must be torch.bfloat16"),
    (dict(cos=torch.zeros(8, 40), sin=torch.zeros(8, 40)), "multiple of 16"), (dict(k_weight=torch.zeros(3)), "norm weights"),
    (dict(q_out=_r(1, 3, 2)), "q_out must be"), (dict(cache=_c(1, 1, 8).expand(1, 2, 8, REC)), "expanded")])
def test_rope_append_refusals(entry, change, match):
    cos, sin = P.table(8, 128)
    _refused(kv4.rope_append, dict(cache=_c(1, 2, 8), q=_r(1, 4, 2), k=_r(1, 2, 2), v=_r(1, 2, 2), cos=cos, sin=sin,
                                   start=_i()), change, match)


@pytest.mark.parametrize("change,match", [
    (dict(T=-1), "T must be"), (dict(k_out=_r(1, 2, 3)), "k_out must be"), (dict(v_out=_r(1, 2, 3)), "v_out must be"),
    (dict(k_out=_r(1, 2, 2, dtype=torch.float16)), "bf16 or fp32"), (dict(start=_i(5)), "start must hold"),
    (dict(k_out=_r(1, 2, 2), v_out=_r(1, 2, 2, dtype=torch.float32)), "v_out must be torch.bfloat16"),
    (dict(v_out=_r(1, 1, 2).expand(1, 2, 2, D)), "expanded")])
def test_unpack_refusals(entry, change, match):
    _refused(kv4.unpack, dict(cache=_c(1, 2, 8), start=_i(), T=2, k_out=_r(1, 2, 2), v_out=_r(1, 2, 2)), change, match)


@pytest.mark.parametrize("change,match", [
    (dict(cache=_c(2, 2, 8)), "same requests"), (dict(cache=_c(1, 3, 8)), "multiple of the KV heads"),
    (dict(cache=_c(1, 8, 8)), "multiple of the KV heads"), (dict(cache=_c(1, 0, 8)), "multiple of the KV heads"),
    (dict(n=None), "n must be given"), (dict(n=_i(2)), "n must hold"), (dict(n=torch.zeros(1)), "n must be"),
    (dict(out=_r(1, 4, 2, dtype=torch.float16)), "bf16 or fp32"), (dict(out=_r(1, 4, 1)), "out must be"),
    (dict(out=_r(1, 4, 2), out_dtype=torch.float32), "out_dtype"),
    (dict(out=_r(1, 1, 2).expand(1, 4, 2, D)), "expanded"),
    (dict(workspace=torch.zeros(4)), "workspace must be"),
    (dict(workspace=torch.zeros(64, dtype=torch.uint8)), "needs a 16-byte aligned workspace of"),
    (dict(q=_r(1, 4, 2).requires_grad_()), "no backward pass")])
def test_decode_attention_refusals(entry, change, match):
    _refused(kv4.decode_attention, dict(q=_r(1, 4, 2), cache=_c(1, 2, 8), n=_i(), out=_r(1, 4, 2),
                                        workspace=torch.zeros(16, dtype=torch.uint8)), change, match)


@pytest.mark.parametrize("change,match", [
    (dict(q=_r(4, dtype=torch.float32)), "q must be"), (dict(q=torch.zeros(4, 64, dtype=BF)), r"\(4, 128\)"),
    (dict(cache=_c(3, 8)), "multiple of the cache's"), (dict(cache=_c(1, 2, 8)), "cache must be"),
    (dict(sel_idx=torch.zeros(4, 2, dtype=torch.int64)), "sel_idx"), (dict(exp_idx=None), "exp_idx"), (dict(exp_idx=torch.zeros(3, 2, dtype=torch.int32)), "exp_idx"),
    (dict(exp_idx=torch.zeros(4, 4, dtype=torch.int32)[:, ::2]), "contiguous"),
    (dict(nb=9), "kbar and vbar must be"), (dict(nb=-1), "bad list sizes"), (dict(vbar=_r(4, 5)), "kbar and vbar"),
    (dict(kbar=_r(3, 6), vbar=_r(3, 6)), "kbar and vbar must be"), (dict(kbar=None, nb=2), "kbar must be|kbar and vbar"),
    (dict(log_n=torch.zeros(4, 4)), "log_n"), (dict(out=torch.zeros(4, 64)), r"\(4, 128\)"),
    (dict(out=_r(1).expand(4, D)), "overlap"), (dict(vbar=_r(4, 6).requires_grad_()), "no backward pass")])
def test_flash_attention_refusals(entry, change, match):
    i = torch.zeros(4, 2, dtype=torch.int32)
    _refused(kv4.flash_attention, dict(q=_r(4), cache=_c(2, 8), sel_idx=i, exp_idx=i, kbar=_r(4, 6), vbar=_r(4, 6),
                                       log_n=torch.zeros(4, 6)), change, match)


def test_blocks_match_the_header():
    """Each packed block has the size and the field kinds of the header's struct."""
    src = open(os.path.join(os.path.dirname(__file__), "..", "include", "openattention_b200.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    structs = {name: body for body, name in re.findall(r"typedef struct \{([^}]*)\} (\w+);", src)}

    def fields(body):
        out = ""
        for decl in (d.strip() for d in body.split(";")):
            if not decl:
                continue
            kind = re.match(r"(?:const )?(\w+)", decl).group(1)
            for name in decl.split(","):
                n = int((re.search(r"\[(\d)\]", name) or [0, 1])[1])
                out += fields(structs[kind]) * n if kind in structs else ("d" if kind == "double" else "q") * n
        return out

    for name, block in _lib.BLOCKS.items():
        flat = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qd])", block.format))
        assert flat == fields(structs[name + "_args"]), name
        assert _lib.load()[name](None, None) == 1 and b"null arguments" in _lib.load().oa_last_error_string()


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
