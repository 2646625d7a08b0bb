"""Build recipe for libvhap_hip.so (gfx950 only).  hipcc cross-compiles without a GPU.

    python -m vhap_amd.build [--force]

The shared library is written IN-TREE (vhap_amd/lib/libvhap_hip.so): it is git-ignored but
travels to the GPU box with the gpurun snapshot.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
LIBDIR = os.path.join(HERE, "lib")
SO = os.path.join(LIBDIR, "libvhap_hip.so")
HOST_SRC = os.path.join(CSRC, "host.cpp")
HOST_SO = os.path.join(LIBDIR, "vhap_host.so")            # extension module over torch's C++ API (no kernels): see csrc/host.cpp
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-munsafe-fp-atomics",
         # no packed-fp32 instructions: the compiler forms them from ordinary float code by itself, and some of their forms have given wrong
         # results on this hardware (the host pass of hipcc does not know the feature and says so: harmless)
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wall", "-Wno-unused-function", f"-I{INCLUDE}", f"-I{CSRC}"]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def _host_command():
    import sysconfig
    import torch
    t = os.path.dirname(torch.__file__)
    return [os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            "-isystem", f"{t}/include", "-isystem", f"{t}/include/torch/csrc/api/include", "-isystem", "/opt/rocm/include",
            "-isystem", sysconfig.get_paths()["include"], f"-I{INCLUDE}", HOST_SRC, "-o", HOST_SO, f"-L{t}/lib", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python"]


def _deps_mtime():
    m = 0.0
    for d in (CSRC, INCLUDE):
        for f in os.listdir(d):
            if f.endswith((".h", ".hip")):
                m = max(m, os.path.getmtime(os.path.join(d, f)))
    return m


def build(force=False, verbose=True):
    os.makedirs(LIBDIR, exist_ok=True)
    hdr_m = max(os.path.getmtime(os.path.join(d, f)) for d in (CSRC, INCLUDE) for f in os.listdir(d) if f.endswith(".h"))
    objs, rebuilt = [], False
    procs = []
    for src in sources():
        obj = os.path.join(LIBDIR, os.path.basename(src)[:-4] + ".o")
        objs.append(obj)
        if force or not os.path.exists(obj) or os.path.getmtime(obj) < max(os.path.getmtime(src), hdr_m):
            cmd = [HIPCC, *FLAGS, "-x", "hip", "-c", src, "-o", obj]
            if verbose:
                print(" ".join(cmd), flush=True)
            procs.append((src, subprocess.Popen(cmd)))
            rebuilt = True
    if force or not os.path.exists(HOST_SO) or os.path.getmtime(HOST_SO) < max(os.path.getmtime(HOST_SRC), hdr_m):
        cmd = _host_command()
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((HOST_SRC, subprocess.Popen(cmd)))
    for src, p in procs:
        if p.wait() != 0:
            raise RuntimeError(f"compiling {src} failed")
    if rebuilt or not os.path.exists(SO):
        cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", SO, *objs]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    return SO


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(SO)
