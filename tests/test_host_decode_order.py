"""fm_moe_decode refuses a call before it launches anything (no GPU needed: a launch would fail
with an error of its own, so the refusal's words show that none was tried)."""

import ctypes as C

import pytest

from nanopysche_amd import _lib

P = C.c_void_p(256)   # passes for an aligned pointer
ODD = C.c_void_p(264)
T, D, K, E = 3, 256, 2, 4


def weights(kind=_lib.DECODE_BF16, H=128, w1=256, w2=256, w3=256, s=None):
    return _lib.FmDecodeWeights(kind, H, w1, w2, w3, s, s, s)


def refused(match, experts=None, shared=None, ld_x=D, norm=None, out=P, out_dtype=0, ld_out=D):
    lib = _lib.load()
    w = experts or weights()
    rc = lib.fm_moe_decode(P, ld_x, T, D, P, 0, D, None, 0, None, norm, 0, 1e-6, E, K, 0, 0, C.byref(w),
                           None if shared is None else C.byref(shared), P, P, out, out_dtype, ld_out, P, 1 << 30, None)
    assert rc != 0 and match in lib.fm_last_error_string(), lib.fm_last_error_string()


@pytest.mark.parametrize("match,kw", [
    (b"bad weight kind", dict(experts=weights(kind=2))),
    (b"weights must be given", dict(experts=weights(w2=None))),
    (b"weights must be given", dict(experts=weights(w3=264))),
    (b"scales", dict(experts=weights(kind=_lib.DECODE_INT8))),
    (b"scales", dict(experts=weights(kind=_lib.DECODE_INT8, s=260))),
    (b"one kind", dict(shared=weights(kind=_lib.DECODE_INT8, s=256))),
    (b"weights must be given", dict(shared=weights(w1=None))),
    (b"multiples of 128", dict(shared=weights(H=0))),
    (b"multiples of 128", dict(experts=weights(H=100))),
    (b"output", dict(out=ODD)),
    (b"output", dict(out_dtype=2)),
    (b"output", dict(ld_out=D - 4)),
    (b"output", dict(ld_out=D + 2)),
    (b"2^23", dict(ld_x=(1 << 23) + 8)),
    (b"output", dict(ld_x=(1 << 23) + 8, norm=P, out=ODD)),   # a normed x is read at a pitch of its own
])
def test_refused_before_the_router_runs(match, kw):
    refused(match, **kw)
