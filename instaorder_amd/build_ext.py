"""Builds libmsda_hip.so and libenc_hip.so in-tree with hipcc for gfx950 (no hipify, no torch cpp_extension)."""
import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SRC = os.path.join(HERE, "csrc", "msda_hip.hip")
LIB = os.path.join(HERE, "libmsda_hip.so")
ENC_SRC = os.path.join(HERE, "csrc", "enc_hip.hip")
ENC_LIB = os.path.join(HERE, "libenc_hip.so")
# packed fp32 instructions off: some of their forms have given wrong results on this hardware
HIPCC_FLAGS = ["-O3", "--offload-arch=gfx950", "-std=c++17", "-shared", "-fPIC",
               "-munsafe-fp-atomics", "-Wall", "-Wextra",
               "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
               "-I" + os.path.join(ROOT, "include")]


def find_hipcc():
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (need ROCm to build libmsda_hip.so)")


def build(force=False, verbose=False):
    """Compiles what is missing or older than its sources (all with force), both libraries at once; returns LIB."""
    csrc, include = os.path.dirname(SRC), os.path.join(ROOT, "include")
    running = []
    for prefix, src, lib in (("msda_", SRC, LIB), ("enc_", ENC_SRC, ENC_LIB)):
        deps = [os.path.join(d, f) for d in (csrc, include) for f in os.listdir(d) if f.startswith(prefix)]
        if (not force and os.path.exists(lib)
                and all(os.path.getmtime(lib) >= os.path.getmtime(d) for d in deps)):
            continue
        cmd = [find_hipcc()] + HIPCC_FLAGS + ["-o", lib, src]
        if verbose:
            print(" ".join(cmd))
        running.append((cmd, subprocess.Popen(cmd)))
    failed = [cmd for cmd, p in running if p.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose=True))
