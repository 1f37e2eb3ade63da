"""Builds libodwscl.so (every HIP kernel + the C-ABI) for gfx950 and _bind.so (torch-side glue in front of it), in-tree.

hipcc cross-compiles without a GPU, so this also runs in the CPU-only build
container; the resulting .so is git-ignored.
"""
import glob
import json
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libodwscl.so")
BIND, BIND_SRC = os.path.join(HERE, "_bind.so"), os.path.join(CSRC, "bind.cpp")
RECORD = os.path.join(HERE, "build", "commands.json")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
# -ffp-contract=off: ROI bin / sample coordinates must round exactly like the
# reference's separate fp32 mul and add; kernels that want FMAs ask for them
# explicitly (fmaf / MFMA).
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
            ["-I" + sysconfig.get_paths()["include"], BIND_SRC, "-o", BIND, "-L" + HERE, "-l:" + os.path.basename(LIB),
             "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_hip", "-Wl,-rpath,$ORIGIN"])


def _object(src):
    return os.path.splitext(src)[0] + ".o"


def _commands():
    """Every output and the command that makes it: an output whose command was another one (other flags, a source that came or went, another
    torch) is as stale as one that is older than its sources."""
    import torch
    cmds = {_object(src): [HIPCC] + FLAGS + ["-c", src, "-o", _object(src)] for src in sources()}
    cmds[LIB] = [HIPCC, "--offload-arch=" + ARCH, "-shared", "-fPIC", "-o", LIB] + [_object(src) for src in sources()]
    cmds[BIND] = _bind_command()
    return cmds, {out: [a.replace(HERE, ".") for a in cmd] + ([torch.__version__] if out == BIND else []) for out, cmd in cmds.items()}


def _recorded():
    try:
        with open(RECORD) as f:
            return json.load(f)
    except (OSError, ValueError):
        return {}


def _record(made):
    os.makedirs(os.path.dirname(RECORD), exist_ok=True)
    with open(RECORD + ".new", "w") as f:
        json.dump(made, f, indent=1, sort_keys=True)
    os.replace(RECORD + ".new", RECORD)


def _stale():
    if not os.path.exists(LIB) or not os.path.exists(BIND):
        return True
    made = _recorded()
    if any(made.get(os.path.basename(out)) != how for out, how in _commands()[1].items()):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(BIND))
    deps = sources() + [BIND_SRC] + glob.glob(os.path.join(CSRC, "*.h")) + \
        glob.glob(os.path.join(HERE, "..", "include", "*.h"))
    return any(os.path.getmtime(p) > t for p in deps)


def build(force=False, verbose=False):
    """Compile csrc/*.hip -> libodwscl.so (objects cached next to the sources), csrc/bind.cpp -> _bind.so."""
    if not force and not _stale():
        return LIB
    cmds, how = _commands()
    name = os.path.basename
    made = {} if force else {name(out): how[out] for out in cmds if out != LIB and _recorded().get(name(out)) == how[out]}
    _record(made)                       # (what is about to be made again is not recorded until it is there)
    procs = []
    for src in sources():
        obj = _object(src)
        newest_dep = max([os.path.getmtime(src)] + [os.path.getmtime(h) for h in
                         glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(HERE, "..", "include", "*.h"))])
        if name(obj) in made and os.path.exists(obj) and os.path.getmtime(obj) > newest_dep:
            continue
        cmd = cmds[obj]
        made.pop(name(obj), None)
        _record(made)
        if verbose:
            print(" ".join(cmd))
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError("hipcc failed on %s:\n%s" % (src, out.decode()))
        if verbose and out:
            print(out.decode())
        made[name(_object(src))] = how[_object(src)]
    subprocess.check_call(cmds[LIB])
    made[name(LIB)] = how[LIB]
    _record(made)
    newest = max(os.path.getmtime(p) for p in [BIND_SRC] + glob.glob(os.path.join(HERE, "..", "include", "*.h")))
    if name(BIND) not in made or not os.path.exists(BIND) or os.path.getmtime(BIND) <= newest:
        if verbose:
            print(" ".join(cmds[BIND]))
        subprocess.check_call(cmds[BIND])
        made[name(BIND)] = how[BIND]
        _record(made)
    else:
        os.utime(BIND)
    return LIB


if __name__ == "__main__":
    import sys
    print(build(force="-f" in sys.argv, verbose=True))
