"""Build libsdfx_hip.so (the C-ABI HIP library) in-tree for gfx950 with hipcc.

    python stable-dreamfusion_amd/build.py [--force] [--verbose] [--devtools]

--devtools builds libsdfx_hip_dev.so instead: the same sources with -DSDFX_DEVTOOLS (implementation switches, measurement
knobs, superseded kernels; include/sdfx_devtools.h). The product library has none of them.

hipcc cross-compiles without a GPU; the resulting .so sits next to the sources (git-ignored,
but shipped to the GPU box with the repository snapshot).
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.normpath(os.path.join(HERE, "..", "include"))
# superseded / measurement-only kernels that only the devtools library compiles in (field_dot2.inc.h, attention_pipe.inc.h): they
# live outside the product source tree
DEVTOOLS_KERNELS = os.path.normpath(os.path.join(HERE, "..", "tools", "devtools_kernels"))
LIB = os.path.join(CSRC, "libsdfx_hip.so")
DEV_LIB = os.path.join(CSRC, "libsdfx_hip_dev.so")
BIND = os.path.join(CSRC, "_sdfx_train.so")      # train_ops_bind.cpp: the training operators as C++ autograd functions (host code only)
SOURCES = ["sdfx_core.hip", "raymarching.hip", "gridencoder.hip", "gridencoder_fwd.hip", "gridencoder_bwd_binned.hip", "encoders.hip", "field.hip", "optim.hip", "shade.hip", "render.hip", "occupancy.hip", "infer.hip", "head.hip", "sds.hip", "dmtet.hip", "raster.hip", "groupnorm.hip", "groupnorm_train.hip", "geglu_train.hip", "conv.hip", "attention.hip", "attention_train.hip", "attention_train_dq.hip", "attention_train_dkdv.hip"]
ARCH = "gfx950"
# -ffp-contract=off: the march / encode arithmetic must not gain FMAs the source does not spell
# out (bit-exact ray counts and fp32 features against the CPU oracle).
# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32. hipcc -O3 forms them from ordinary float code, and some of their forms have given
# wrong results on MI355X now and then; the scalar instructions round the same way, so no result changes. (The host pass warns that
# it does not know the feature: harmless.)
FLAGS = ["--offload-arch=" + ARCH, "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-fno-fast-math",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wall", "-Wno-unused-function", "-Wno-pass-failed", "-I", INCLUDE]


def hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found: the HIP extension cannot be built")
    return exe


def _deps_mtime(devtools: bool = False) -> float:
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")] + [os.path.join(INCLUDE, "sdfx.h")]
    hdrs.append(os.path.abspath(__file__))       # (the flags)
    if devtools and os.path.isdir(DEVTOOLS_KERNELS):
        hdrs += [os.path.join(DEVTOOLS_KERNELS, f) for f in os.listdir(DEVTOOLS_KERNELS) if f.endswith(".h")]
    return max(os.path.getmtime(h) for h in hdrs)


def _compile(src: str, force: bool, verbose: bool, devtools: bool = False) -> str:
    path = os.path.join(CSRC, src)
    obj = os.path.join(CSRC, "build_dev" if devtools else "build", src.replace(".hip", ".o"))
    os.makedirs(os.path.dirname(obj), exist_ok=True)
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(path), _deps_mtime(devtools)):
        return obj
    cmd = [hipcc()] + FLAGS + (["-DSDFX_DEVTOOLS", "-I", DEVTOOLS_KERNELS] if devtools else []) + ["-c", path, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return obj


def _build_bind(force: bool, verbose: bool) -> str:
    """train_ops_bind.cpp against the installed torch, with the host compiler. It holds no kernel and does not link the HIP library: _sdfx.py
    hands it the entry points of the library it opened."""
    src = os.path.join(CSRC, "train_ops_bind.cpp")
    newest = max(os.path.getmtime(f) for f in (src, os.path.join(INCLUDE, "sdfx.h"), os.path.abspath(__file__)))
    if not force and os.path.exists(BIND) and os.path.getmtime(BIND) >= newest:
        return BIND
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    inc = [a for p in (*cpp_extension.include_paths(), sysconfig.get_paths()["include"], "/opt/rocm/include") for a in ("-isystem", p)]
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           "-DTORCH_EXTENSION_NAME=_sdfx_train", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *inc, src, "-o", BIND,
           "-L" + os.path.join(os.path.dirname(torch.__file__), "lib"), "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return BIND


def build(force: bool = False, verbose: bool = False, devtools: bool = False) -> str:
    sources = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    lib = DEV_LIB if devtools else LIB
    with cf.ThreadPoolExecutor(max_workers=min(len(sources), os.cpu_count() or 1)) as ex:
        bind = None if devtools else ex.submit(_build_bind, force, verbose)          # (one for both libraries)
        objs = list(ex.map(lambda s: _compile(s, force, verbose, devtools), sources))
    if bind is not None:
        bind.result()
    if force or not os.path.exists(lib) or os.path.getmtime(lib) < max(os.path.getmtime(o) for o in objs):
        cmd = [hipcc(), "--offload-arch=" + ARCH, "-shared", "-fPIC", "-o", lib] + objs
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    return lib


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv or "-v" in sys.argv, devtools="--devtools" in sys.argv))
