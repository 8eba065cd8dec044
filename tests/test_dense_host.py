"""The library of the products on 16-bit weights on the host (no GPU): its exports and structs are what the header says, its entry
points refuse bad arguments before any launch, and the built code keeps the wait states of its matrix instructions."""
import ctypes
import os
import re
import subprocess

import pytest

from eva_amd import _lib
from tests import test_isa_hazards

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "evamx_dense.h")
FAKE = 0x10000


def test_exports():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(evamx_[a-z0-9_]+)\s*\(", text))
    assert names == set(_lib.DENSE_EXPORTS)
    assert _lib.dense_lib().evamx_dense_version() == _lib.DENSE_VERSION


@pytest.mark.parametrize("name,cls", [("evamx_linear_args", _lib.LinearArgs), ("evamx_linear_grad_args", _lib.LinearGradArgs)])
def test_struct_layout(tmp_path, name, cls):
    fields = [f for f, _ in cls._fields_]
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "evamx_dense.h"', 'int main(void) {',
             f'printf("%zu\\n", sizeof({name}));', *(f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields), "return 0; }"]
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def _call(cls, fn, **kw):
    a = dict.fromkeys((f for f, _ in cls._fields_), 0)
    a.update(x=FAKE, w=FAKE, workspace=FAKE, workspace_bytes=1 << 40, x_stride=64, w_stride=64, w_expert_stride=64 * 32, dtype=1, rows=8,
             n_in=64, n_out=32, experts=1)
    a.update(dict(y=FAKE, y_stride=32) if cls is _lib.LinearArgs else dict(grad=FAKE, grad_x=FAKE, grad_w=FAKE, grad_bias=FAKE, grad_stride=32,
                                                                            grad_x_stride=64))
    a.update(kw)
    rc = fn(ctypes.byref(cls(*(a[f] for f, _ in cls._fields_))), None)
    assert rc == 0 or _lib.dense_lib().evamx_dense_last_error()
    return rc


SIZES = [dict(rows=-1), dict(rows=(1 << 24) + 1), dict(n_in=0), dict(n_out=0), dict(n_in=(1 << 18) + 1), dict(n_out=(1 << 18) + 1),
         dict(experts=0), dict(experts=2), dict(experts=1025, starts=FAKE), dict(dtype=2), dict(dtype=-1), dict(act=5), dict(act=-1),
         dict(act=4, n_out=31), dict(limit=1.0), dict(act=4, limit=-1.0), dict(act=4, limit=float("nan")), dict(x_stride=63), dict(w_stride=63),
         dict(experts=2, starts=FAKE, w_expert_stride=2047)]


@pytest.mark.parametrize("bad", SIZES + [dict(x=0), dict(w=0), dict(y=0), dict(y_stride=31), dict(residual=FAKE, residual_stride=31),
                                         dict(rows=100, n_in=4096, x_stride=4096, w_stride=4096, workspace=0),
                                         dict(rows=100, n_in=4096, x_stride=4096, w_stride=4096, workspace=FAKE + 8)])
def test_linear_refuses(bad):
    assert _call(_lib.LinearArgs, _lib.dense_lib().evamx_linear, **bad) == _lib.EVAMX_EINVAL


@pytest.mark.parametrize("bad", SIZES + [dict(grad=0), dict(x=0), dict(w=0), dict(act=1, pre=0), dict(grad_stride=31), dict(grad_x_stride=63),
                                         dict(act=1, pre=FAKE, workspace=0), dict(act=1, pre=FAKE, workspace=FAKE + 4)])
def test_gradient_refuses(bad):
    assert _call(_lib.LinearGradArgs, _lib.dense_lib().evamx_linear_grad, **bad) == _lib.EVAMX_EINVAL


def test_null_and_sizes():
    L = _lib.dense_lib()
    assert L.evamx_linear(None, None) == _lib.EVAMX_EINVAL and L.evamx_linear_grad(None, None) == _lib.EVAMX_EINVAL
    assert _call(_lib.LinearArgs, L.evamx_linear, rows=0, x=0, w=0, y=0) == _lib.EVAMX_OK                  # nothing to do
    wide = dict(rows=100, n_in=4096, x_stride=4096, w_stride=4096)
    assert _call(_lib.LinearArgs, L.evamx_linear, workspace_bytes=64, **wide) == _lib.EVAMX_ENOSPACE
    assert _call(_lib.LinearGradArgs, L.evamx_linear_grad, act=1, pre=FAKE, workspace_bytes=64) == _lib.EVAMX_ENOSPACE
    assert L.evamx_linear_workspace_bytes(100, 4096, 32, 1, 0, 1) > 0 and L.evamx_linear_workspace_bytes(100, 0, 32, 1, 0, 1) == 0
    # what a larger call's workspace serves stays within what was asked for, at any size
    for rows in (0, 1, 64, 65, 1000, 1 << 24):
        for n in (1, 520, 1 << 18):
            assert L.evamx_linear_grad_workspace_bytes(rows, n, 64, 1, 0, 1, 0) < (1 << 45)


def test_built_library_keeps_the_wait_states(tmp_path, monkeypatch):
    """As tests/test_isa_hazards.py for libevamx.so, with the bf16 instruction, whose passes are the fp16 one's."""
    if not os.path.exists(test_isa_hazards.OBJDUMP):
        pytest.skip("no llvm-objdump")
    monkeypatch.setattr(test_isa_hazards, "WAITS", {**test_isa_hazards.WAITS, "v_mfma_f32_16x16x32_bf16": test_isa_hazards.WAITS["v_mfma_f32_16x16x32_f16"]})
    lib = tmp_path / "lib.so"
    lib.write_bytes(open(_lib.DENSE_LIB_PATH, "rb").read())
    subprocess.run([test_isa_hazards.OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, capture_output=True, check=True)
    objects = sorted(p for p in os.listdir(tmp_path) if p.endswith("gfx950"))
    assert len(objects) >= 3
    count, bad = 0, []
    for o in objects:
        for name, code in test_isa_hazards._functions(tmp_path / o):
            count += sum(t.startswith("v_mfma") for _, t, _ in code)
            bad += [(name,) + v for v in test_isa_hazards._violations(code)]
    assert count > 1000 and not bad, (len(bad), bad[:8])
