"""Build the C-ABI HIP libraries in-tree for gfx950 with hipcc.

    python -m eva_amd.build            # csrc/*.hip -> eva_amd/libevamx.so, csrc/dense/*.hip -> eva_amd/libevamx_dense.so

Objects go to eva_amd/_build/ (git-ignored); the .so files sit next to this file so that they travel
with the source tree.
"""
from __future__ import annotations

import concurrent.futures
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libevamx.so")
DENSE_CSRC = os.path.join(CSRC, "dense")
DENSE_LIB = os.path.join(HERE, "libevamx_dense.so")
ARCH = "gfx950"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-fno-gpu-rdc",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function", "-Wno-unused-variable",
]


def sources(folder: str = CSRC):
    return sorted(os.path.join(folder, f) for f in os.listdir(folder) if f.endswith(".hip"))


def _compile(src):
    obj = os.path.join(OBJ, os.path.relpath(src, CSRC)[:-4].replace(os.sep, "_") + ".o")
    cmd = [HIPCC, *FLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    msgs = "\n".join(l for l in (r.stdout + r.stderr).splitlines()
                     if "packed-fp32-ops" not in l)   # host pass: feature unknown to x86, harmless
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{msgs}")
    return obj, msgs


def _link(lib, objs):
    tmp = lib + ".tmp"
    r = subprocess.run([HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs,
                        "-Wl,-rpath,/opt/rocm/lib"], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}{r.stderr}")
    os.replace(tmp, lib)


def build(verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    main, dense = sources(), sources(DENSE_CSRC)
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        results = list(ex.map(_compile, main + dense))
    if verbose:
        for _, m in results:
            if m.strip():
                print(m, file=sys.stderr)
    objs = [o for o, _ in results]
    _link(LIB, objs[:len(main)])
    _link(DENSE_LIB, objs[len(main):])
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
