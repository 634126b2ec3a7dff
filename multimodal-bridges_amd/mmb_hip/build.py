"""In-tree build of libmmb_hip.so (hipcc, gfx950 only).  `python -m mmb_hip.build` or
__graft_entry__.build().  Rebuilds only when a source is newer than the library."""
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "csrc")
LIB = os.path.join(HERE, os.environ.get("MMB_LIB_NAME", "libmmb_hip.so"))      # developer builds: other name
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# max-memory-clause: the fused kernels live on the 256-VGPR limit; this pre-RA strategy spills less there (S3 generation
# kernel 168 -> 144 B/lane of scratch, S2 112 -> 68, training forward 392 -> 316) and measured +2..5 % on every bench
# line
# no packed float arithmetic: some of its forms have given wrong results on this machine without an error
FLAGS = ["-O3", "--offload-arch=gfx950", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wall", "-Wno-unused-function",
         "-Wno-unused-variable", "-Wno-unused-but-set-variable"]
SCHED = os.environ.get("MMB_SCHED", "max-memory-clause")                       # developer A/B: MMB_SCHED=default
if SCHED != "default":
    FLAGS += ["-mllvm", "-amdgpu-sched-strategy=" + SCHED]
FLAGS += os.environ.get("MMB_EXTRA_FLAGS", "").split()


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=True):
    srcs = sources()
    hdrs = glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "..", "..", "include", "*.h"))
    objs = []
    procs = []
    objdir = os.path.join(CSRC, "build" + os.environ.get("MMB_OBJ_SUFFIX", ""))
    os.makedirs(objdir, exist_ok=True)
    for s in srcs:
        o = os.path.join(objdir, os.path.basename(s)[:-4] + ".o")
        objs.append(o)
        deps = [s] + hdrs
        if s.endswith("_w5.hip"):                       # a second compilation of another source (#include "....hip")
            deps.append(s[:-7] + ".hip")
        if force or _stale(o, deps):
            cmd = [HIPCC] + FLAGS + ["-c", s, "-o", o]
            if verbose:
                print(" ".join(cmd), flush=True)
            procs.append((s, subprocess.Popen(cmd)))
    for s, p in procs:
        if p.wait() != 0:
            raise RuntimeError(f"hipcc failed on {s}")
    if force or procs or _stale(LIB, objs):
        cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB)
