"""Builds csrc/*.hip into libadcdiff.so (gfx950 only) next to this file.

hipcc cross-compiles without a GPU, so this runs in the CPU-only build container; the resulting
shared object travels to the GPU box with the source tree.
"""
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libadcdiff.so")
BINDING = os.path.join(HERE, "libadcdiff_torch.so")    # csrc/torch_binding.cpp: host code only, against the installed torch
SOURCES = [("gemm.hip", []), ("gemm_tr.hip", []), ("elementwise.hip", ["-ffp-contract=off"]), ("unet.hip", []), ("train.hip", []),
           ("residual_norm.hip", []), ("grad_norm.hip", []), ("gemm_i8.hip", [])]
# packed float32 instructions stay off: some of their forms have given wrong results on this hardware now and then
COMMON = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-Wall", "-Wno-unused-function",
          "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build_library(force=False, verbose=False):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    # the assembly main loop of the 4-wave GEMM is generated (register-allocated by hand in the generator)
    gen, inc = os.path.join(CSRC, "gen_w4_mainloop.py"), os.path.join(CSRC, "w4_mainloop.inc")
    if force or _stale(inc, [gen]):
        subprocess.run([sys.executable, gen, inc], check=True)
    inc_i8 = os.path.join(CSRC, "w4_mainloop_i8.inc")
    if force or _stale(inc_i8, [gen]):
        subprocess.run([sys.executable, gen, "--i8", inc_i8], check=True)
    # this file among them: it holds the flags, and objects of other flags must not be linked
    headers = [os.path.abspath(__file__), inc_i8, os.path.join(CSRC, "common.h"), os.path.join(CSRC, "row_access.h"), os.path.join(CSRC, "unet_plan.h"), inc, os.path.join(os.path.dirname(HERE), "include", "adcdiff.h")]
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    objs, cmds = [], []
    for src, extra in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(objdir, src.replace(".hip", ".o"))
        if force or _stale(o, [s] + headers):
            cmds.append([hipcc] + COMMON + extra + ["-c", s, "-o", o])
            if verbose:
                print(" ".join(cmds[-1]))
        objs.append(o)
    with ThreadPoolExecutor(max_workers=4) as pool:      # one compiler per stale source, four at a time
        for done in [pool.submit(subprocess.run, cmd, check=True) for cmd in cmds]:
            done.result()
    if force or _stale(LIB, objs):
        cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
    build_binding(force, verbose)
    return LIB


def build_binding(force=False, verbose=False):
    """The PyTorch operators over the C ABI; the adcdiff_* symbols are resolved from libadcdiff.so when it is loaded."""
    src = os.path.join(CSRC, "torch_binding.cpp")
    import torch
    from torch.utils import cpp_extension
    deps = [os.path.abspath(__file__), src, os.path.join(os.path.dirname(HERE), "include", "adcdiff.h"), torch.__file__]
    if force or _stale(BINDING, deps):
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
               "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI, "-I/opt/rocm/include"]
        cmd += ["-I" + p for p in cpp_extension.include_paths()] + [src, "-o", BINDING]
        cmd += ["-L" + p for p in cpp_extension.library_paths()] + ["-ltorch", "-ltorch_cpu", "-lc10", "-lc10_hip"]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
    return BINDING


if __name__ == "__main__":
    print(build_library(verbose=True))
