"""Build libneumesh_hip.so for gfx950 with hipcc (in-tree, next to the sources).

hipcc cross-compiles without a GPU, so this runs in the build container; the resulting .so is
git-ignored but travels to the GPU box with the repository snapshot.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import tempfile

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc")
LIB_PATH = os.path.join(CSRC, "libneumesh_hip.so")
# the same sources with -DNM_TESTING: the product's exports + test hooks (host octree build, octree export, scalar-ALU self-check
# of the MFMA tile code, phase stamps).  Loaded by a few tests and by the measurement tools only -- never by the package.
TESTING_LIB_PATH = os.path.join(os.path.dirname(os.path.dirname(CSRC)), "tests", "_build", "libneumesh_hip_testing.so")
SOURCES = ["nm_api.hip", "nm_dense.hip", "nm_scan.hip"]   # one translation unit each, compiled in parallel
HEADERS = sorted(f for f in os.listdir(CSRC) if f.endswith((".h", ".inc"))) + [os.path.join("..", "..", "include", "neumesh_hip.h")]
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off", "-fPIC", "-shared",
         "-Wno-unused-value",
         # no packed fp32 instructions (v_pk_add_f32, ...): some of their forms have given wrong results on this hardware.  (The host pass does not know
         # the feature and says so: harmless.)
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _stale(path: str) -> bool:
    if not os.path.exists(path):
        return True
    t = os.path.getmtime(path)
    return any(os.path.getmtime(os.path.join(CSRC, f)) > t for f in SOURCES + HEADERS)


def _compile(path: str, extra, verbose: bool) -> str:
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        raise RuntimeError("hipcc not found: cannot build " + os.path.basename(path))
    os.makedirs(os.path.dirname(path), exist_ok=True)
    with tempfile.TemporaryDirectory() as tmp:
        objects = [os.path.join(tmp, os.path.splitext(s)[0] + ".o") for s in SOURCES]
        flags = [f for f in FLAGS if f != "-shared"]
        cmds = [[hipcc, *flags, *extra, "-c", os.path.join(CSRC, s), "-o", o] for s, o in zip(SOURCES, objects)]
        link = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", *objects, "-o", path + ".tmp"]
        if verbose:
            print("\n".join(" ".join(c) for c in cmds + [link]))
        procs = [subprocess.Popen(c, cwd=CSRC) for c in cmds]
        codes = [p.wait() for p in procs]
        for c, code in zip(cmds, codes):
            if code != 0:
                raise subprocess.CalledProcessError(code, c)
        subprocess.check_call(link, cwd=CSRC)
    os.replace(path + ".tmp", path)
    return path


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the HIP library if it is missing or older than its sources. Returns its path."""
    if not force and not _stale(LIB_PATH):
        return LIB_PATH
    return _compile(LIB_PATH, [], verbose)


def build_testing(force: bool = False, verbose: bool = False) -> str:
    """The test / measurement build (-DNM_TESTING) under tests/_build/.  Returns its path."""
    if not force and not _stale(TESTING_LIB_PATH):
        return TESTING_LIB_PATH
    return _compile(TESTING_LIB_PATH, ["-DNM_TESTING"], verbose)


if __name__ == "__main__":
    print(build(force=True, verbose=True))
    print(build_testing(force=True, verbose=True))
