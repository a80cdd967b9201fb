"""Build libtecogan_hip.so in-tree with hipcc for gfx950 (no JIT cache: the .so travels with the repo)."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libtecogan_hip.so")
SOURCES = ["conv_igemm.hip", "conv3x3.hip", "conv3x3_ws.hip", "conv3x3_dma.hip", "conv3x3_wr.hip", "conv4x4s2.hip", "resblock_lat.hip", "resblock_chain.hip", "resblock_plane.hip", "resblock_thr.hip", "hr_bwd_lat.hip", "hr_fwd_lat.hip", "conv_wgrad.hip", "conv_wgrad_tr.hip", "warp.hip", "pointwise.hip", "schedule.hip", "losses.hip", "runtime.hip"]
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-munsafe-fp-atomics", "-Wno-unused-result"]
# No v_pk_{add,mul,fma}_f32: the compiler forms them from ordinary float code at -O3, and some of their operand forms have given
# wrong results on MI355X now and then (the host pass does not know the feature and says so: harmless).  The older sources keep
# the instruction selection that their frozen deterministic results were recorded with: with this flag one gradient's error
# against the fp64 oracle moved by 4 % (tests/golden/c3_det_max_norm.json holds it to 2 %).
SCALAR_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
SCALAR_FP32_SOURCES = ["gated_norm.hip", "gated_scan.hip", "fp8_quantize.hip", "fp8_matmul.hip"]
SOURCES += SCALAR_FP32_SOURCES


def flags_for(src):
    """The compiler flags of one source."""
    return FLAGS + (SCALAR_FP32 if src in SCALAR_FP32_SOURCES else [])


def _newer(a, b):
    return (not os.path.exists(b)) or os.path.getmtime(a) > os.path.getmtime(b)


def build(force=False, verbose=True):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    deps = [os.path.join(CSRC, "common.h"), os.path.join(CSRC, "handoff.h"), os.path.join(CSRC, "fp8.h"), os.path.join(HERE, "..", "include", "tecogan_hip.h")]
    objs, procs = [], []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(CSRC, src.replace(".hip", ".o"))
        objs.append(o)
        if force or _newer(s, o) or any(_newer(d, o) for d in deps):
            cmd = [hipcc] + flags_for(src) + ["-c", s, "-o", o]
            if verbose:
                print(" ".join(cmd), flush=True)
            procs.append((src, subprocess.Popen(cmd)))
    for src, p in procs:
        if p.wait() != 0:
            raise RuntimeError("hipcc failed on " + src)
    if force or procs or not os.path.exists(LIB) or any(_newer(o, LIB) for o in objs):
        cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
