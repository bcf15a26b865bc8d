"""Builds libmsda_hip.so and libenc_hip.so in-tree with hipcc for gfx950 (no hipify), and with g++ the binding of the
latter (host code against torch's headers)."""
import os
import shutil
import subprocess
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SRC = os.path.join(HERE, "csrc", "msda_hip.hip")
LIB = os.path.join(HERE, "libmsda_hip.so")
ENC_SRC = os.path.join(HERE, "csrc", "enc_hip.hip")
ENC_LIB = os.path.join(HERE, "libenc_hip.so")
BIND_SRC = os.path.join(HERE, "csrc", "enc_bind.cpp")
BIND_LIB = os.path.join(HERE, "_enc_bind.so")
# packed fp32 instructions off: some of their forms have given wrong results on this hardware
HIPCC_FLAGS = ["-O3", "--offload-arch=gfx950", "-std=c++17", "-shared", "-fPIC",
               "-munsafe-fp-atomics", "-Wall", "-Wextra",
               "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
               "-I" + os.path.join(ROOT, "include")]


def bind_commands():
    """(compile, link) of the binding; the object can be compiled while the library it links with is."""
    import torch
    base = os.path.dirname(torch.__file__)
    include = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
               os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include")]
    obj = os.path.join(HERE, "_enc_bind.o")
    compile_ = ["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
                "-DTORCH_EXTENSION_NAME=_enc_bind", "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI,
                "-I" + os.path.join(ROOT, "include"), *["-isystem" + d for d in include],
                "-isystem" + sysconfig.get_paths()["include"], "-c", "-o", obj, BIND_SRC]
    link = ["g++", "-shared", "-o", BIND_LIB, obj, "-L" + HERE, "-lenc_hip", "-L" + os.path.join(base, "lib"), "-ltorch",
            "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip", "-Wl,-rpath,$ORIGIN"]
    return compile_, link


def find_hipcc():
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (need ROCm to build libmsda_hip.so)")


def build(force=False, verbose=False):
    """Compiles what is missing or older than its sources (all with force), side by side; returns LIB."""
    csrc, include = os.path.dirname(SRC), os.path.join(ROOT, "include")

    def stale(lib, deps):
        return force or not os.path.exists(lib) or any(os.path.getmtime(lib) < os.path.getmtime(d) for d in deps)

    def start(cmd):
        if verbose:
            print(" ".join(cmd))
        return cmd, subprocess.Popen(cmd)

    def finish(started):
        failed = [cmd for cmd, p in started if p.wait() != 0]
        if failed:
            raise subprocess.CalledProcessError(1, failed[0])

    running = []
    for prefix, src, lib in (("msda_", SRC, LIB), ("enc_", ENC_SRC, ENC_LIB)):
        deps = [os.path.join(d, f) for d in (csrc, include) for f in os.listdir(d) if f.startswith(prefix) and not f.endswith(".cpp")]
        if stale(lib, deps):
            running.append(start([find_hipcc()] + HIPCC_FLAGS + ["-o", lib, src]))
    bind = stale(BIND_LIB, [BIND_SRC, os.path.join(include, "enc_hip.h")])
    if bind:
        compile_, link = bind_commands()
        running.append(start(compile_))
    finish(running)
    if bind:
        finish([start(link)])
        os.remove(compile_[-2])
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose=True))
