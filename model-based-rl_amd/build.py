"""Build the native code in-tree: csrc/models_gen.hpp (generated), csrc/libmbrl_hip.so (hipcc, gfx950) and
csrc/optim_bind.so (g++: the argument lists of optim.py, which are Python lists of tensors)."""
import os
import shutil
import subprocess
import sysconfig

from . import compile_planar

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(CSRC, "libmbrl_hip.so")
BIND = os.path.join(CSRC, "optim_bind.so")
SOURCES = ["mbrl_hip.hip", "planar_lean.hpp", "wave_or.hpp", "models_gen.hpp", "abi_error.hpp", "optim.hip"]


def _hipcc():
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("hipcc not found")


def needs_build():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, s) for s in SOURCES] + [os.path.join(HERE, "modelspec.py"),
                                                       os.path.join(HERE, "compile_planar.py"),
                                                       os.path.abspath(__file__),       # the compiler flags live here
                                                       os.path.join(HERE, "..", "include", "mbrl.h")]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


# No packed float32 instructions: some of their forms have been seen to give wrong results.  (The host pass of hipcc warns that
# it does not know the feature.)
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

# -pragma-unroll-threshold: the tree-sparse factorisation must unroll completely (register arrays);
# -disable-machine-licm: loop-invariant integer bookkeeping must not be hoisted into 100+ registers;
# no-NaN / no-infinity / no-signed-zero arithmetic: lets x * 0.0 and x + 0.0 fold (model tables are full of zeros)
# and drops the canonicalisation before min / max; non-finite results are still caught, by a test on the bits
# (t_finite in planar_lean.hpp) that these flags cannot fold away.
HIPCC_FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wno-pass-failed",
               "-mllvm", "-pragma-unroll-threshold=1000000", "-mllvm", "-disable-machine-licm",
               "-mllvm", "-amdgpu-use-amdgpu-trackers=1",   # GCN register-pressure trackers in the scheduler: ~30 % fewer AGPR copies
               "-mllvm", "-amdgpu-sched-strategy=max-ilp",  # occupancy is pinned at one wave per SIMD anyway: schedule for
                                                            # latency, not for registers (-2.7 %; iterative-ilp, minreg slower)
               "-fno-honor-nans", "-fno-honor-infinities", "-fno-signed-zeros"] + NO_PACKED_FP32


# The optimiser-step operators are a translation unit of their own: they promise IEEE results for infinities and NaN, which
# the flags above give away, and gain nothing from that schedule.
OPTIM_FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC"] + NO_PACKED_FP32


def compile_lib(out, extra_flags=()):
    """csrc/mbrl_hip.hip (with `extra_flags`: the profiling tools make their variants with it) and csrc/optim.hip -> `out`."""
    objs = [out + ".main.o", out + ".optim.o"]
    jobs = [subprocess.Popen([_hipcc()] + flags + ["-c", "-o", obj, os.path.join(CSRC, src)], cwd=CSRC)
            for obj, src, flags in ((objs[0], "mbrl_hip.hip", HIPCC_FLAGS + list(extra_flags)), (objs[1], "optim.hip", OPTIM_FLAGS))]
    if any([j.wait() for j in jobs]):
        raise RuntimeError("hipcc failed")
    subprocess.check_call([_hipcc(), "--offload-arch=gfx950", "-shared", "-o", out + ".tmp"] + objs, cwd=CSRC)
    for obj in objs:
        os.remove(obj)
    os.replace(out + ".tmp", out)
    return out


def build_bind(force=False):
    """csrc/optim_bind.cpp -> csrc/optim_bind.so: a CPython module over torch's C++ tensors (host code only)."""
    src, deps = os.path.join(CSRC, "optim_bind.cpp"), [os.path.join(CSRC, "optim_bind.cpp"), os.path.join(HERE, "..", "include", "mbrl.h")]
    if not force and os.path.exists(BIND) and all(os.path.getmtime(d) <= os.path.getmtime(BIND) for d in deps):
        return BIND
    import torch
    from torch.utils import cpp_extension
    rocm = os.path.dirname(os.path.dirname(_hipcc()))
    inc = cpp_extension.include_paths() + [sysconfig.get_paths()["include"], os.path.join(rocm, "include")]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch.compiled_with_cxx11_abi(),
           "-D__HIP_PLATFORM_AMD__=1"]        # the HIP runtime's headers ask a plain host compiler for it
    cmd += ["-isystem" + d for d in inc] + ["-o", BIND + ".tmp", src, "-L" + libs, "-ltorch_python", "-ltorch_cpu", "-lc10_hip", "-lc10"]
    subprocess.check_call(cmd, cwd=CSRC)
    os.replace(BIND + ".tmp", BIND)
    return BIND


def build_hip(force=False, verbose=False):
    """hipcc --offload-arch=gfx950 -> csrc/libmbrl_hip.so (cross-compiles without a GPU)."""
    compile_planar.write_header()
    if not force and not needs_build():
        return LIB
    return compile_lib(LIB, ["-Rpass-analysis=kernel-resource-usage"] if verbose else [])
