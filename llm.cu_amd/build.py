"""Build libllmt.so (all HIP kernels + the C ABI) and the llm_train driver.

Compiles every source under csrc/ with hipcc for gfx950 into _build/, links
libllmt.so next to this file, then links the llm_train executable against it.
Always recompiles (the CPU-side "does it build" check relies on that).

    python llm.cu_amd/build.py [-j N] [-v]
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
CSRC = HERE / "csrc"
BUILD = HERE / "_build"
LIB = HERE / "libllmt.so"
TRAIN = HERE / "llm_train"

ARCH = "gfx950"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# The packed-fp32 feature is disabled for every device compile: hipcc -O3
# otherwise forms v_pk_*_f32 from plain float code on gfx950.
CFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-fPIC", "-std=c++20", "-Wall", "-Wno-unused-function",
    "-Wno-unused-variable", "-Wno-unused-but-set-variable",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{ROOT / 'include'}", f"-I{CSRC}",
]


def _sources():
    return sorted(list(CSRC.glob("*.hip")) + list(CSRC.glob("*.cpp")))


# Per-file additions.  attn.hip, packed_fwd.hip (the attention forwards): MFMA results and
# accumulators in ordinary VGPRs (its softmax works on every score, so AGPR
# copies cost VALU slots).  The backward (attn_bwd.hip) keeps its dK/dV
# accumulators in AGPRs.
EXTRA = {"attn.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
         "packed_fwd.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"]}


def _compile(src: Path, verbose: bool) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [HIPCC, *CFLAGS, *EXTRA.get(src.name, []), "-c", str(src), "-o", str(obj)]
    if src.suffix == ".cpp":
        cmd[1:1] = ["-x", "hip"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    out = "\n".join(l for l in (r.stdout + r.stderr).splitlines()
                    if "packed-fp32-ops" not in l)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{out}")
    if verbose and out.strip():
        print(out)
    return obj


def build(jobs: int = 8, verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    srcs = _sources()
    with cf.ThreadPoolExecutor(max_workers=max(1, jobs)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp),
           *map(str, objs)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n" + r.stdout + r.stderr)
    os.replace(tmp, LIB)
    drv = HERE / "llm_train.cpp"
    if drv.exists():
        cmd = [HIPCC, "-O2", "-std=c++17", f"-I{ROOT / 'include'}", str(drv), "-o", str(TRAIN),
               f"-L{HERE}", "-lllmt", "-Wl,-rpath,$ORIGIN"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("llm_train link failed:\n" + r.stdout + r.stderr)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("-j", type=int, default=min(8, os.cpu_count() or 1))
    ap.add_argument("-v", action="store_true")
    a = ap.parse_args()
    print(build(a.j, a.v))
