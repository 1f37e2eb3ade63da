"""Builds libodwscl.so (every HIP kernel + the C-ABI) for gfx950 and _bind.so (torch-side glue in front of it), in-tree.

hipcc cross-compiles without a GPU, so this also runs in the CPU-only build
container; the resulting .so is git-ignored but ships with gpurun snapshots.
"""
import glob
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libodwscl.so")
BIND, BIND_SRC = os.path.join(HERE, "_bind.so"), os.path.join(CSRC, "bind.cpp")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
# -ffp-contract=off: ROI bin / sample coordinates must round exactly like the
# reference's separate fp32 mul and add (SURVEY.md s7 hard part vii); kernels
# that want FMAs ask for them explicitly (fmaf / MFMA).
# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 -- the compiler forms them from ordinary float code, and some of their
# forms have given wrong results on this hardware now and then (hipcc's host pass warns that it does not know the feature).
FLAGS = ["--offload-arch=" + ARCH, "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
         "-fvisibility=hidden", "-Wall", "-Wno-unused-function",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


# experiment builds (tools/exp, timing studies that knowingly produce wrong results): ODW_EXTRA_FLAGS="-DODW_EXPERIMENTS"
FLAGS += [f for f in os.environ.get("ODW_EXTRA_FLAGS", "").split() if f]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def _bind_command():
    """Host code only: the C++ compiler, torch's headers and the HIP headers that those include."""
    import sysconfig
    import torch
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), "/opt/rocm/include"]
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
             "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch.compiled_with_cxx11_abi())] + [f for i in inc for f in ("-isystem", i)] +
            ["-I" + sysconfig.get_paths()["include"], BIND_SRC, "-o", BIND, "-L" + HERE, "-l:" + os.path.basename(LIB), "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu",
             "-ltorch", "-lc10", "-lc10_hip", "-Wl,-rpath,$ORIGIN"])


def _stale():
    if not os.path.exists(LIB) or not os.path.exists(BIND):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(BIND))
    deps = sources() + [BIND_SRC] + glob.glob(os.path.join(CSRC, "*.h")) + \
        glob.glob(os.path.join(HERE, "..", "include", "*.h"))
    return any(os.path.getmtime(p) > t for p in deps)


def build(force=False, verbose=False):
    """Compile csrc/*.hip -> libodwscl.so (objects cached next to the sources), csrc/bind.cpp -> _bind.so."""
    if not force and not _stale():
        return LIB
    objs = []
    procs = []
    for src in sources():
        obj = os.path.splitext(src)[0] + ".o"
        objs.append(obj)
        newest_dep = max([os.path.getmtime(src)] + [os.path.getmtime(h) for h in
                         glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(HERE, "..", "include", "*.h"))])
        if not force and os.path.exists(obj) and os.path.getmtime(obj) > newest_dep:
            continue
        cmd = [HIPCC] + FLAGS + ["-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd))
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError("hipcc failed on %s:\n%s" % (src, out.decode()))
        if verbose and out:
            print(out.decode())
    cmd = [HIPCC, "--offload-arch=" + ARCH, "-shared", "-fPIC", "-o", LIB] + objs
    subprocess.check_call(cmd)
    newest = max(os.path.getmtime(p) for p in [BIND_SRC] + glob.glob(os.path.join(HERE, "..", "include", "*.h")))
    if force or not os.path.exists(BIND) or os.path.getmtime(BIND) <= newest:
        cmd = _bind_command()
        if verbose:
            print(" ".join(cmd))
        subprocess.check_call(cmd)
    else:
        os.utime(BIND)
    return LIB


if __name__ == "__main__":
    import sys
    print(build(force="-f" in sys.argv, verbose=True))
