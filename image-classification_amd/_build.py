"""Build libmi_knn.so (gfx950) in-tree with hipcc.  Cross-compiles without a GPU."""
from __future__ import annotations

import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmi_knn.so")
COMMON = ["host_common.h", os.path.join("..", "..", "include", "mi_knn.h")]
# translation units and the headers that each one includes
SOURCES = {
    "mi_knn.hip": ["sim_kernel.h", "sim_walk_kernel.h", "select_kernel.h", "vote_kernel.h", "moco_kernel.h"] + COMMON,
    "mi_cache.hip": ["cache_kernel.h"] + COMMON,
}
# packed fp32 instructions stay out of the device code: some of their forms have given wrong results on this part, without an error
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: cannot build libmi_knn.so")


def _newer(target: str, deps) -> bool:
    """Whether one of `deps` is newer than `target`, or `target` is not there."""
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in deps)


def _paths(source: str):
    return [os.path.join(CSRC, f) for f in [source] + SOURCES[source]]


def is_stale() -> bool:
    return any(_newer(LIB, _paths(s)) for s in SOURCES)


def build(force: bool = False, verbose: bool = False) -> str:
    """One object file for each translation unit, compiled side by side, linked into one library."""
    if not force and not is_stale():
        return LIB
    cc, objects, running = _hipcc(), [], []
    for source in SOURCES:
        obj = os.path.join(CSRC, os.path.splitext(source)[0] + ".o")
        objects.append(obj)
        if force or _newer(obj, _paths(source)):
            cmd = [cc] + FLAGS + ["-c", os.path.join(CSRC, source), "-o", obj]
            if verbose:
                cmd.append("-Rpass-analysis=kernel-resource-usage")
            running.append((cmd, subprocess.Popen(cmd, cwd=CSRC)))
    codes = [(cmd, p.wait()) for cmd, p in running]
    for cmd, code in codes:
        if code:
            raise subprocess.CalledProcessError(code, cmd)
    subprocess.check_call([cc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objects, cwd=CSRC)
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose=True))
