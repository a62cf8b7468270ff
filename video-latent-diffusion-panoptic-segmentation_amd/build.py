"""Build the gfx950 HIP library (lib/libldmseg_hip.so) and its torch binding (lib/ldmseg_torch.so) in-tree.

    python video-latent-diffusion-panoptic-segmentation_amd/build.py [--force] [--jobs N]

hipcc cross-compiles for gfx950 without a GPU, so this runs in the CPU container and the
resulting .so travels to the GPU box with the repo snapshot.  Objects are rebuilt only
when their source, a shared header or this file (the flags) is newer.
"""
import argparse
import concurrent.futures as cf
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "build")
LIB_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIB_DIR, "libldmseg_hip.so")
BINDING = os.path.join(LIB_DIR, "ldmseg_torch.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
CFLAGS = ["-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}", "-Wall", "-Wno-unused-function",
          "-Wno-unused-variable", "-I" + os.path.join(ROOT, "include"),
          # no packed fp32 arithmetic (v_pk_{add,mul,fma}_f32): some of its forms have given wrong results on this
          # card.  hipcc's host pass warns that it does not know the feature
          "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _headers():
    return glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(ROOT, "include", "*.h"))


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src, obj):
    cmd = [HIPCC, *CFLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def build_binding(force=False, verbose=True):
    """The C++ torch binding (csrc/torch_binding.cpp): host code, linked against torch's own libraries."""
    src = os.path.join(CSRC, "torch_binding.cpp")
    if not force and not _stale(BINDING, [src, *_headers(), os.path.abspath(__file__)]):
        return BINDING
    import sysconfig

    import torch
    if verbose:
        print("[build] compiling the torch binding", flush=True)
    inc, lib = (os.path.join(os.path.dirname(torch.__file__), d) for d in ("include", "lib"))
    rocm = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DUSE_ROCM",
           "-D__HIP_PLATFORM_AMD__", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I" + inc,
           "-I" + sysconfig.get_paths()["include"], "-I" + rocm, src, "-o", BINDING + ".tmp", "-L" + lib, "-lc10",
           "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"torch binding failed:\n{r.stdout}\n{r.stderr}")
    os.replace(BINDING + ".tmp", BINDING)
    return BINDING


def build(force=False, jobs=None, verbose=True):
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    build_binding(force, verbose)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    hdrs = _headers()
    objs, todo = [], []
    for s in srcs:
        o = os.path.join(BUILD, os.path.basename(s)[:-4] + ".o")
        objs.append(o)
        if force or _stale(o, [s, *hdrs, os.path.abspath(__file__)]):
            todo.append((s, o))
    jobs = jobs or min(8, os.cpu_count() or 1, max(1, len(todo)))
    if todo:
        if verbose:
            print(f"[build] compiling {len(todo)} HIP sources for {ARCH} ({jobs} jobs)", flush=True)
        with cf.ThreadPoolExecutor(jobs) as ex:
            list(ex.map(lambda so: _compile(*so), todo))
    if force or todo or _stale(LIB, objs):
        cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", LIB + ".tmp"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(LIB + ".tmp", LIB)
        if verbose:
            print(f"[build] linked {LIB}", flush=True)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    a = ap.parse_args()
    try:
        build(a.force, a.jobs)
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
