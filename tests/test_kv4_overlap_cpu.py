"""Written tensors whose elements share memory are refused before any launch: overlaps of one dim with itself (expanded
tensors, small strides) and of dims with each other (two strides that reach the same rows).  Views that only look
unusual are not."""
import pytest
import torch

from test_kv4_cpu import _c, _i, _r, _refused, entry  # noqa: F401 (entry: a fixture)
import kv4_plain as P
from openattention_b200 import kv4, rotary

D, REC, BF = 128, 144, torch.bfloat16


def _view(sizes, strides, dtype=BF):
    n = 1 + sum((s - 1) * abs(t) for s, t in zip(sizes, strides))
    return torch.zeros(n, dtype=dtype).as_strided(sizes, strides)


# (B, heads, T, 128): strides under which two (b, h, t) are the same row, or overlap
SHARED = [(512, 512, 128), (256, 256, 128), (128, 256, 128), (128, 2048, 128), (384, 256, 128), (2048, 160, 128), (0, 256, 128)]


@pytest.mark.parametrize("st", SHARED)
def test_rows_that_overlap_across_dims(entry, st):  # noqa: F811
    cos, sin = P.table(8, 128)
    out = _view((2, 4, 2, D), (*st, 1))
    q, k = _r(2, 4, 2), _r(2, 2, 2)
    _refused(rotary.qk_norm_rope, dict(q=q, k=k, cos=cos, sin=sin, start=_i(), q_out=out), {}, "q_out.*overlap")
    _refused(rotary.qk_norm_rope, dict(q=k, k=q, cos=cos, sin=sin, start=_i(), k_out=out), {}, "k_out.*overlap")
    _refused(kv4.rope_append, dict(cache=_c(2, 2, 8), q=q, k=k, v=k, cos=cos, sin=sin, start=_i(), q_out=out), {}, "q_out.*overlap")
    _refused(kv4.unpack, dict(cache=_c(2, 4, 8), start=_i(), T=2, k_out=out, v_out=_r(2, 4, 2)), {}, "k_out.*overlap")
    _refused(kv4.unpack, dict(cache=_c(2, 4, 8), start=_i(), T=2, k_out=_r(2, 4, 2), v_out=out), {}, "v_out.*overlap")
    _refused(kv4.decode_attention, dict(q=q, cache=_c(2, 2, 8), n=_i(), out=out, workspace=torch.zeros(16, dtype=torch.uint8)), {},
             "out.*overlap")


RUN = 8 * REC


@pytest.mark.parametrize("st", [(RUN, RUN), (2 * RUN, 2 * RUN), (4 * RUN, 2 * RUN), (-RUN, RUN), (3 * RUN - 16, RUN),
                                (2 * RUN, RUN - 144)])
def test_caches_that_share_records_across_dims(entry, st, monkeypatch):  # noqa: F811
    """(B, hkv) = (2, 3) heads of 8 records; a negative stride cannot be made with torch, so the fields are given."""
    monkeypatch.setattr(kv4, "_cache", lambda c, ndim=4: (c.data_ptr(), 2, 3, 8, REC, *st, REC, 1))
    cos, sin = P.table(8, 128)
    k = _r(2, 3, 2)
    _refused(kv4.append, dict(cache=_c(2, 3, 8), k=k, v=k, start=_i()), {}, "share records")
    _refused(kv4.rope_append, dict(cache=_c(2, 3, 8), q=k, k=k, v=k, cos=cos, sin=sin, start=_i()), {}, "share records")


def _passes_the_checks(call, **a):
    """The call gets as far as the launch, which fails where there is no GPU (fixture `entry`)."""
    from test_kv4_cpu import _fake
    with pytest.raises(RuntimeError, match="CUDA|driver|device"):
        call(**{n: _fake(t) for n, t in a.items()})


def test_views_that_do_not_overlap_are_taken(entry):  # noqa: F811
    cos, sin = P.table(8, 128)
    q, k = _r(2, 4, 3), _r(2, 2, 3)
    big = _r(3, 5, 8, 4)                                          # (3, 5, 8, 4, 128)
    for out in (big[:2, :4, :3, 0], big[1:, ::2, 1:5, 2].transpose(1, 2)[:, :4, :3], _r(3, 2, 4).permute(1, 2, 0, 3),
                _r(4, 3, 2).permute(2, 0, 1, 3), _view((2, 4, 3, D), (128, 8192, 1024, 1))):
        _passes_the_checks(rotary.qk_norm_rope, q=q, k=k, cos=cos, sin=sin, start=_i(), q_out=out)
    one = _view((2, 4, 1, D), (2048, 128, 0, 1))                  # the stride of a dim of one element counts for nothing
    _passes_the_checks(rotary.qk_norm_rope, q=_r(2, 4, 1), k=_r(2, 2, 1), cos=cos, sin=sin, start=_i(), q_out=one)
    for cache in (_c(3, 5, 8)[1:, ::2][:, :2], _c(2, 2, 8).transpose(0, 1), _c(2, 2, 20)[:, :, 4:12]):
        _passes_the_checks(kv4.append, cache=cache, k=k, v=k, start=_i())
