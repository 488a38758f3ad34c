"""In-tree build of libtagpipe_hip.so (HIP kernels + C ABI) for gfx950.

hipcc cross-compiles without a GPU.  The library is written next to the
sources so that it travels with the tree; it is never installed elsewhere.
Beside it stands the torch module of the reply calls (_tp_torch.so), where
there is a torch to build it against.
"""
import concurrent.futures
import importlib.util
import os
import runpy
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libtagpipe_hip.so")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
HIPCC = os.environ.get("HIPCC", os.path.join(ROCM, "bin", "hipcc"))

SOURCES = ["tp_kernels.hip", "tp_reply.hip", "tp_api.cpp", "tp_tables.cpp", "tp_grammar.cpp"]
HEADERS = ["tp_common.h", "tp_pipeline.h", "tp_fast.h", "tp_lean.h", "tp_launch.h", "tp_reply.h", "tp_grammar.hpp", "tp_tables.hpp", "tp_json.hpp", "tp_case_tables.inc",
           os.path.join("..", "..", "include", "tagpipe.h")]
# -ffp-contract=off: the score arithmetic (1.0 - i * 0.01) must round like the reference's, with no fused multiply-add.
COMMON = ["-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-Wall", "-Wno-unused-function"]
# Two 32-bit float operations in one instruction are left out: some forms of them have given wrong results on these GPUs.
DEVICE = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


# The torch side of the reply calls: a Python module against the torch that is installed, host code only.
TORCH_SOURCES = ["tp_torch.cpp", os.path.join("..", "..", "include", "tagpipe.h")]
TORCH_LIB = os.path.join(HERE, "_tp_torch.so")
CXX = os.environ.get("CXX", "g++")


def _torch_module_missing():
    """Why the torch module cannot be built here, or None.  The C library does without it (a C# program needs nothing else); the reply calls of
    replies.py say so when one is made."""
    spec = importlib.util.find_spec("torch")                    # without importing it
    if spec is None or not spec.origin:
        return "torch is not installed"
    if not os.path.isdir(os.path.join(os.path.dirname(spec.origin), "include", "torch", "csrc")):
        return "torch is installed without its headers"
    if shutil.which(CXX) is None:
        return "there is no C++ compiler %s" % CXX
    return None


def _torch_name():
    """The installed torch, as `torch.__version__ torch.version.git_version`, without importing it."""
    spec = importlib.util.find_spec("torch")
    v = runpy.run_path(os.path.join(os.path.dirname(spec.origin), "version.py"))
    return "%s %s" % (v["__version__"], v["git_version"])


def _build_torch_module(verbose):
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    cmd = [CXX, '-DTP_TORCH_NAME="%s"' % _torch_name(), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-fvisibility=hidden", "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI,
           "-I" + sysconfig.get_paths()["include"]]
    for d in ("include", os.path.join("include", "torch", "csrc", "api", "include")):
        cmd += ["-isystem", os.path.join(root, d)]
    cmd += [os.path.join(CSRC, TORCH_SOURCES[0]), "-o", TORCH_LIB, "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)


def _older(lib, sources):
    return not os.path.exists(lib) or any(os.path.getmtime(os.path.join(CSRC, f)) > os.path.getmtime(lib) for f in sources)


def _stale():
    return _older(LIB, SOURCES + HEADERS)


def _torch_module_stale():
    if _older(TORCH_LIB, TORCH_SOURCES):
        return True
    with open(TORCH_LIB, "rb") as f:                             # it names the torch it was built against (its layouts are compiled in)
        return ("torch module for " + _torch_name()).encode() + b"\0" not in f.read()


def build(force=False, verbose=False, prof=False):
    """prof=True builds the diagnostic variant libtagpipe_hip_prof.so (per-section cycle counters inside k_fast)."""
    if prof:
        return _build(LIB.replace(".so", "_prof.so"), "_prof.o", ["-DTP_PROF"], verbose)
    variant = os.environ.get("TAGPIPE_BUILD_VARIANT")          # experiments: "name:-Dflag,-Dflag" -> libtagpipe_hip_name.so
    if variant:
        name, flags = variant.split(":", 1)
        return _build(LIB.replace(".so", "_%s.so" % name), "_%s.o" % name, [f for f in flags.split(",") if f], verbose, kernels_only=True)
    missing = _torch_module_missing()
    if missing and (force or verbose):
        print("%s: the library is built without the torch module of the reply calls" % missing, flush=True)
    with concurrent.futures.ThreadPoolExecutor(1) as beside:
        torch_module = beside.submit(_build_torch_module, verbose) if not missing and (force or _torch_module_stale()) else None
        if force or _stale():
            _build(LIB, ".o", [], verbose)
        if torch_module:
            torch_module.result()
    return LIB


def _build(lib, obj_suffix, extra, verbose, kernels_only=False):
    objs, cmds = [], []
    for src in SOURCES:
        obj = os.path.join(CSRC, os.path.splitext(src)[0] + obj_suffix)
        if kernels_only and not src.endswith(".hip"):       # experiments only touch the kernels: reuse the main build's host objects
            objs.append(os.path.join(CSRC, os.path.splitext(src)[0] + ".o"))
            continue
        cmd = [HIPCC, "--offload-arch=gfx950"] + COMMON + extra
        if src.endswith(".hip"):
            cmd += ["-x", "hip"] + DEVICE
        else:
            cmd += ["-x", "c++", "-D__HIP_PLATFORM_AMD__", "-I" + os.path.join(ROCM, "include")]
        cmds.append(cmd + ["-c", os.path.join(CSRC, src), "-o", obj])
        if verbose:
            print(" ".join(cmds[-1]), flush=True)
        objs.append(obj)
    with concurrent.futures.ThreadPoolExecutor(len(cmds)) as pool:                 # the kernels' two files take a minute each
        list(pool.map(subprocess.check_call, cmds))
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-o", lib] + objs
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return lib


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, prof="--prof" in sys.argv)
