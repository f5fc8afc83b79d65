"""Launches that the shared prefix attention plans for (no GPU: the plan is the host's)."""
import ctypes

import pytest


def launches(groups, r, hq, hkv, shared, own, sink=0, recent=0, arrivals=4096, **kw):
    from heterokv import _lib
    s = _lib.SharedArgs(group=r, shared_blocks=shared // 16, arrivals=arrivals)
    d = s.decode
    d.batch, d.num_q_heads, d.num_kv_heads, d.head_dim = groups * r, hq, hkv, 128
    d.int4_max_len, d.int4_lens = shared + own, 4096
    for n in (sink, recent):
        if n:
            d.f16[d.num_f16_zones].max_len, d.f16[d.num_f16_zones].capacity = n, -(-n // 16) * 16
            d.num_f16_zones += 1
    for k, v in kw.items():
        setattr(d, k, v)
    return _lib.load().hkv_shared_launches(ctypes.byref(s))


@pytest.mark.parametrize("case,want", [
    (dict(groups=1, r=2, hq=32, hkv=8, shared=1024, own=17, sink=16, recent=64), 1),
    (dict(groups=1, r=2, hq=32, hkv=8, shared=1024, own=17, sink=16, recent=64, arrivals=0), 2),
    (dict(groups=1, r=5, hq=32, hkv=8, shared=1024, own=17), 2),        # two row tiles
    (dict(groups=1, r=2, hq=32, hkv=8, shared=28608, own=200), 2),      # long
    (dict(groups=1, r=3, hq=32, hkv=8, shared=160, own=1, num_kv_heads=7), 0),
    (dict(groups=1, r=3, hq=32, hkv=8, shared=160, own=1, int4_max_len=100), 0)])
def test_launches(case, want):
    assert launches(**case) == want


def test_null():
    from heterokv import _lib
    assert _lib.load().hkv_shared_launches(None) == 0 and b"null" in _lib.load().hkv_last_error()
