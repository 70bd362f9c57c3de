"""Builds conformer_amd/libfcenc_hip.so from csrc/*.hip with hipcc for gfx950 (in-tree).

    python -m conformer_amd.build [--force]

hipcc cross-compiles without a GPU, so this runs in the build container; the resulting .so
travels to the GPU box with the tree.  Nothing is compiled at import time.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(CSRC, "build")
LIB = os.path.join(HERE, "libfcenc_hip.so")
SOURCES = ["api.hip", "gemm.hip", "conv256.hip", "conv12.hip", "conv3p.hip", "ffn.hip", "ffn_wide.hip", "convmod.hip", "convmod_wide.hip", "elementwise.hip", "attention.hip",
           "stream.hip", "decode.hip", "mel.hip", "train.hip", "pages.hip", "page_attn.hip", "sample.hip"]
# No packed fp32 instructions (v_pk_add / mul / fma_f32): hipcc -O3 forms them by itself from ordinary float code, and some
# of their forms have given wrong results now and then.  (The host pass does not know the feature and says so; harmless.)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=fast", "-Wall",
         "-Wno-unused-function", "-Wno-unused-variable", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
# per-file additions.  Without packed fp32 instructions -O3 still groups neighbouring scalar code of these files in its own way.
# elementwise.hip: conv1 is paced by the SiLU of its 655 M outputs, and was faster without the grouping while that still formed
# v_pk_mul_f32 (280.5 -> 275.6 us on MI355X, same bits); the block kernels measured no difference.
EXTRA_FLAGS = {"elementwise.hip": ["-fno-slp-vectorize"], "conv12.hip": ["-fno-slp-vectorize"], "conv3p.hip": ["-fno-slp-vectorize"]}


def _hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found; cannot build libfcenc_hip.so")
    return exe


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _commands(hipcc: str):
    """(source, object, command) of every file."""
    for src in SOURCES:
        s, o = os.path.join(CSRC, src), os.path.join(OBJ, src.replace(".hip", ".o"))
        yield s, o, [hipcc, *FLAGS, *EXTRA_FLAGS.get(src, []), "-c", s, "-o", o]


def _built_with(o: str):
    """The command that made an object, None if that is not known."""
    try:
        with open(o + ".cmd") as f:
            return f.read()
    except OSError:
        return None


def build_native(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    hipcc = _hipcc()
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")]
    headers.append(os.path.join(os.path.dirname(HERE), "include", "fcenc.h"))
    # an object is as old as its sources and its command: changed flags make it again too
    jobs = [(o, cmd) for s, o, cmd in _commands(hipcc) if force or _stale(o, [s] + headers) or _built_with(o) != " ".join(cmd)]

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("hipcc failed:\n" + " ".join(cmd) + "\n" + r.stdout + r.stderr)
        if verbose and r.stderr.strip():
            print(r.stderr, file=sys.stderr)

    def compile_one(job):
        o, cmd = job
        run(cmd)
        with open(o + ".cmd", "w") as f:
            f.write(" ".join(cmd))

    with ThreadPoolExecutor(max_workers=4) as ex:
        list(ex.map(compile_one, jobs))
    objs = [os.path.join(OBJ, s.replace(".hip", ".o")) for s in SOURCES]
    if force or jobs or _stale(LIB, objs):
        run([hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", LIB])
    return LIB


if __name__ == "__main__":
    print(build_native(force="--force" in sys.argv, verbose=True))
