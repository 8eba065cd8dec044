"""Operators on 4-bit weights on the host (no GPU): sizes, and the C ABI's refusals before any launch."""
import ctypes

import pytest

from eva_amd import _lib

FAKE = 0x10000      # never dereferenced: every call below fails validation first


def _weight(**kw):
    d = dict(codes=FAKE, scales=FAKE, zeros=None, count=1, n_out=256, n_in=512, group=128, scale_dtype=_lib.DTYPE_F16)
    d.update(kw)
    return _lib.W4Desc(*[d[f] for f, _ in _lib.W4Desc._fields_])


def test_stored_groups_and_sizes():
    L = _lib.lib()
    assert [L.evamx_w4_stored_group(g) for g in (32, 64, 96, 128, 160, 192, 256, 384, 1024)] == [32, 64, 32, 128, 32, 64, 128, 128, 128]
    assert [L.evamx_w4_stored_group(g) for g in (0, -32, 16, 33, 48)] == [0] * 5
    assert L.evamx_w4_code_bytes(1, 16, 128) == 1024 and L.evamx_w4_code_bytes(3, 17, 129) == 3 * 4 * 1024
    assert L.evamx_w4_group_count(1, 16, 128, 128) == 64 and L.evamx_w4_group_count(2, 17, 513, 32) == 2 * 2 * 2 * 256
    big = _lib.W4_MAX_DIM
    assert L.evamx_w4_code_bytes(1024, big, big) == 1024 * big * big // 2       # sizes do not wrap at 32 bits
    for bad in ((0, 16, 16), (1025, 16, 16), (1, 0, 16), (1, 16, 0), (1, big + 1, 16), (1, 16, big + 1)):
        assert L.evamx_w4_code_bytes(*bad) == 0 and L.evamx_w4_group_count(*bad, 32) == 0
    assert L.evamx_w4_group_count(1, 16, 16, 96) == 0


@pytest.mark.parametrize("bad", [dict(codes=0), dict(scales=0), dict(count=0), dict(n_out=0), dict(n_in=0), dict(n_in=(1 << 18) + 1),
                                 dict(group=96), dict(scale_dtype=2), dict(codes=FAKE + 4), dict(scales=FAKE + 2), dict(zeros=FAKE + 1)])
def test_weights_are_checked(bad):
    L, w = _lib.lib(), _weight(**bad)
    assert L.evamx_w4_dequant(ctypes.byref(w), FAKE, None) == _lib.EVAMX_EINVAL
    assert L.evamx_w4_linear(FAKE, 0, 512, 1, ctypes.byref(w), None, FAKE, 256, FAKE, 1 << 30, None) == _lib.EVAMX_EINVAL
    assert L.evamx_last_error()


def test_pack_is_checked():
    L = _lib.lib()
    for args in ((0, FAKE, None, 128), (FAKE, 0, None, 128), (FAKE, FAKE, FAKE, 128), (FAKE, FAKE, None, 64), (FAKE, FAKE, None, 100)):
        assert L.evamx_w4_pack(*args, ctypes.byref(_weight()), None) == _lib.EVAMX_EINVAL, args
    assert L.evamx_w4_pack(FAKE, FAKE, None, 128, ctypes.byref(_weight(zeros=FAKE)), None) == _lib.EVAMX_EINVAL
    assert L.evamx_w4_dequant(ctypes.byref(_weight()), None, None) == _lib.EVAMX_EINVAL


def test_linear_is_checked():
    L = _lib.lib()
    good = dict(x=FAKE, dt=1, xs=512, rows=4, w=_weight(), bias=None, y=FAKE, ys=256, ws=FAKE, nb=1 << 30)

    def call(**kw):
        a = {**good, **kw}
        return L.evamx_w4_linear(a["x"], a["dt"], a["xs"], a["rows"], ctypes.byref(a["w"]), a["bias"], a["y"], a["ys"], a["ws"], a["nb"], None)

    for bad in (dict(x=0), dict(y=0), dict(ws=0), dict(dt=2), dict(xs=511), dict(ys=255), dict(rows=0), dict(rows=65537),
                dict(w=_weight(count=2)), dict(ws=FAKE + 8)):
        assert call(**bad) == _lib.EVAMX_EINVAL, bad
        assert L.evamx_last_error()
    assert call(nb=16) == _lib.EVAMX_ENOSPACE
    sizes = [L.evamx_w4_linear_workspace_bytes(r, 512) for r in (1, 2, 16, 17, 65536)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > 0
    assert L.evamx_w4_linear_workspace_bytes(0, 512) == 0 and L.evamx_w4_linear_workspace_bytes(65537, 512) == 0
