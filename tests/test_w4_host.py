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
    assert L.evamx_w4_group_count(1, 16, 128, 128) == 16 and L.evamx_w4_group_count(2, 17, 513, 32) == 2 * 2 * 5 * 64
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
    sizes = [L.evamx_w4_linear_workspace_bytes(r, 512) for r in (*range(1, 70), 65536)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] > 0
    assert L.evamx_w4_linear_workspace_bytes(0, 512) == 0 and L.evamx_w4_linear_workspace_bytes(65537, 512) == 0


def _moe(**kw):
    w = {n: _weight(count=9, n_out=o, n_in=i) for n, o, i in (("gate", 256, 512), ("up", 256, 512), ("down", 512, 256))}
    for n in ("gate", "up", "down"):
        for f, v in kw.pop(n, {}).items():
            setattr(w[n], f, v)
    a = _lib.W4MoeArgs(x=FAKE, sel=FAKE, weights=FAKE, gate=ctypes.pointer(w["gate"]), up=ctypes.pointer(w["up"]),
                       down=ctypes.pointer(w["down"]), out=FAKE, workspace=FAKE, workspace_bytes=1 << 40, x_stride=512, out_stride=512,
                       first_expert=0, x_dtype=1, rows=4, topk=2, n_shared=1, limit=10.0)
    for f, v in kw.items():
        setattr(a, f, v)
    return _lib.lib().evamx_w4_moe_forward(ctypes.byref(a), None)


@pytest.mark.parametrize("bad", [
    dict(x=0), dict(sel=0), dict(weights=0), dict(out=0), dict(workspace=0), dict(workspace=FAKE + 4), dict(x_stride=511), dict(out_stride=511),
    dict(x_dtype=2), dict(rows=0), dict(rows=21846), dict(topk=0), dict(topk=33), dict(n_shared=-1), dict(n_shared=10), dict(limit=-1.0),
    dict(limit=float("inf")), dict(limit=float("nan")), dict(gate=dict(codes=0)), dict(up=dict(group=48)), dict(down=dict(n_out=500)),
    dict(up=dict(n_out=255)), dict(down=dict(count=8)), dict(up=dict(group=64)), dict(up=dict(zeros=FAKE)), dict(up=dict(scale_dtype=1)), dict(down=dict(scale_dtype=5)),
])
def test_moe_is_checked(bad):
    assert _moe(**bad) == _lib.EVAMX_EINVAL
    assert _lib.lib().evamx_last_error()


def test_moe_workspace():
    L = _lib.lib()
    assert _moe(workspace_bytes=1000) == _lib.EVAMX_ENOSPACE
    assert L.evamx_w4_moe_forward(None, None) == _lib.EVAMX_EINVAL
    sizes = [L.evamx_w4_moe_workspace_bytes(r, 8, 1, 7168, 2048) for r in (1, 2, 16, 17, 512, 7281)]
    assert sizes[0] > 0 and all(a <= b for a, b in zip(sizes, sizes[1:]))
    for shape in ((8, 1, 64, 64), (32, 32, 64, 32), (1, 0, 7168, 2048), (32, 0, 128, 4096)):       # a larger call's serves a smaller one
        need = [L.evamx_w4_moe_workspace_bytes(r, *shape) for r in (*range(1, 40), 64, 100, 500, 1000)]
        assert all(0 < a <= b for a, b in zip(need, need[1:])), shape
    for bad in ((0, 8, 1, 64, 64), (7282, 8, 1, 64, 64), (1, 0, 0, 64, 64), (1, 8, 33, 64, 64), (1, 8, 0, 0, 64), (1, 8, 0, 64, 1 << 19)):
        assert L.evamx_w4_moe_workspace_bytes(*bad) == 0, bad


@pytest.mark.parametrize("hidden, inter", [(7168, 2048), (100, 16384), (4096, 16300), (64, 1 << 18), (1 << 18, 128), (1 << 18, 1 << 18)])
@pytest.mark.parametrize("topk, shared", [(1, 0), (8, 1), (32, 32)])
def test_the_module_splits_by_every_limit(hidden, inter, topk, shared):
    """The rows of a call that W4Experts makes are within its limits, and no more would be."""
    from eva_amd.w4 import _moe_call_rows
    need, n = _lib.lib().evamx_w4_moe_workspace_bytes, _moe_call_rows(topk + shared, hidden, inter)
    assert n >= 1 and need(n, topk, shared, hidden, inter) > 0 and need(n + 1, topk, shared, hidden, inter) == 0


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    structs = {"evamx_w4_weight": _lib.W4Desc, "evamx_w4_moe_args": _lib.W4MoeArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "evamx.h"', 'int main(void) {']
    for st, cls in structs.items():
        lines.append(f'printf("{st} size %zu\\n", sizeof({st}));')
        lines += [f'printf("{st} {f} %zu\\n", offsetof({st}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(l.rsplit(" ", 1) for l in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for st, cls in structs.items():
        assert int(got[f"{st} size"]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f"{st} {f}"]) == getattr(cls, f).offset, (st, f)
