"""Build librmem_hip.so (gfx950) in-tree with hipcc.  No JIT cache: the .so travels
with the repository snapshot to the GPU box."""
from __future__ import annotations

import os
import subprocess
import sys

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc")
LIB = os.path.join(CSRC, "librmem_hip.so")
SOURCES = ["linear.hip", "read64.hip", "mha.hip", "pointwise.hip", "postproc.hip", "batch.hip", "bank8.hip", "bank8_attn.hip"]
HEADERS = ["rmem_common.h", "bank8.h", "gemm_core.h", "linear_stream.h", "attn_common.h", "launch.h", os.path.join("..", "..", "include", "rmem_hip.h")]


# mha.hip: VGPR form of every MFMA (no AGPRs: the 32x32 score and output tiles are read and written by
# the softmax VALU code, so the accumulator form costs a v_accvgpr move per element and s_nops in
# front of each; 128 registers instead of 128 + 32 also give 4 waves per SIMD instead of 3)
EXTRA_FLAGS = {"mha.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
               # read64.hip: no SLP vectorisation -- it turns the eight per-lane softmax updates into <8 x float>
               # operations whose splat operands (the row reference m, eight copies) it then spills; every reload is a
               # compiler-visible vector-memory access that drains the hand-counted V-fragment ring (s_waitcnt vmcnt(0))
               "read64.hip": ["-fno-slp-vectorize"]}
# No packed fp32 arithmetic (v_pk_add / mul / fma_f32) in any kernel: some of its forms have given wrong results on gfx950 now and
# then.  (The host pass warns that it does not know the feature.)
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _commands() -> list:
    """Every compile command and the link, in order."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    objs = [os.path.join(CSRC, src.replace(".hip", ".o")) for src in SOURCES]
    cmds = [[hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-c", os.path.join(CSRC, src), "-o", obj] +
            NO_PACKED_FP32 + EXTRA_FLAGS.get(src, []) + os.environ.get("RMEM_HIPCC_FLAGS", "").split() for src, obj in zip(SOURCES, objs)]
    return cmds + [[hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs]


def _stamp() -> str:
    """The commands as the library keeps them beside itself (flags decide about its results as sources do), without where they ran."""
    return "\n".join(" ".join(c) for c in _commands()).replace(CSRC + os.sep, "")


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    if any(os.path.getmtime(os.path.join(CSRC, f)) > t for f in SOURCES + HEADERS):
        return True
    try:
        with open(LIB + ".cmd") as f:
            return f.read() != _stamp()
    except OSError:
        return True


def build_lib(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return LIB
    for cmd in _commands():
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.check_call(cmd)
    with open(LIB + ".cmd", "w") as f:
        f.write(_stamp())
    return LIB


if __name__ == "__main__":
    print(build_lib(force="--force" in sys.argv, verbose=True))
