#!/usr/bin/env python3
"""Build libdm_hip.so (gfx950) in-tree with hipcc.  No cmake/ninja; one object per .hip file,
compiled in parallel, linked into diffusion_model_amd/libdm_hip.so."""
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
OUT = os.path.join(PKG, "libdm_hip.so")
OBJ = os.path.join(HERE, "build")
FLAGS = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-ffast-math", "-fno-gpu-rdc",
         "-Wno-unused-result", "-DNDEBUG",
         # no SLP vectorizer: it pairs scalar fp32 adds/muls into v_pk_*_f32, which issue slower than the two
         # scalar ops they replace next to MFMA/exp streams (measured on the attention kernels)
         "-fno-slp-vectorize",
         # no packed fp32 instructions at all: vector types make them without the SLP vectorizer too (the training step takes
         # the same time without them, 14.8 to 15.0 ms)
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
# Sources whose kernels see infinities and NaN in earnest (masked keys, empty rows) or reduce angles in 64 bits: no fast math.
PRECISE = {"dm_cross_fwd.hip", "dm_cross_bwd.hip", "dm_cross_few.hip", "dm_cross_one.hip", "dm_cross_onebwd.hip", "dm_cross_rowsbwd.hip", "dm_rope.hip"}


def hipcc():
    return shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def _compile(src, force=False):
    obj = os.path.join(OBJ, os.path.basename(src) + ".o")
    deps = [src] + [os.path.join(HERE, f) for f in os.listdir(HERE) if f.endswith(".h")] + [
        os.path.join(os.path.dirname(PKG), "include", "dm_hip.h")]
    if not force and os.path.exists(obj) and all(os.path.getmtime(obj) > os.path.getmtime(d) for d in deps):
        return obj, ""
    extra = ["-fno-fast-math"] if os.path.basename(src) in PRECISE else []
    r = subprocess.run([hipcc(), *FLAGS, *extra, "-c", src, "-o", obj], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{r.stdout}\n{r.stderr}")
    return obj, r.stderr


def build(verbose=False, force=False):
    """``force``: compile every source, also where an up-to-date object is there."""
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(os.path.join(HERE, f) for f in os.listdir(HERE) if f.endswith(".hip"))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        res = list(ex.map(lambda src: _compile(src, force), srcs))
    objs = [o for o, _ in res]
    if verbose:
        for _, err in res:
            if err.strip():
                print(err)
    if not force and os.path.exists(OUT) and all(os.path.getmtime(OUT) > os.path.getmtime(o) for o in objs):
        return OUT
    r = subprocess.run([hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", OUT, *objs],
                       capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    return OUT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
