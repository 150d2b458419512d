"""Build the in-tree HIP shared library (gfx950 only).  hipcc cross-compiles without a GPU."""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
SRC = os.path.join(PKG_DIR, "csrc", "lora_kernels.hip")
SRCS = [SRC, os.path.join(PKG_DIR, "csrc", "vit_kernels.hip"), os.path.join(PKG_DIR, "csrc", "loss_kernels.hip"),
        os.path.join(PKG_DIR, "csrc", "fp8_kernels.hip"), os.path.join(PKG_DIR, "csrc", "seg_kernels.hip"),
        os.path.join(PKG_DIR, "csrc", "seq_rows.hip"), os.path.join(PKG_DIR, "csrc", "seq_attention.hip")]
INCLUDE = os.path.join(REPO_DIR, "include")
LIB_NAME = "libsam3_lora_amd.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)


# packed-fp32-ops off: some forms of the packed fp32 instructions that hipcc makes of ordinary float code have given wrong
# results on this hardware now and then; the scalar forms round the same way
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (set HIPCC or install ROCm)")


def needs_build() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    # every source the library is compiled from: the .hip units, the .inc files they include, the public headers
    deps = SRCS + sorted(glob.glob(os.path.join(PKG_DIR, "csrc", "*.inc"))) + sorted(glob.glob(os.path.join(INCLUDE, "*.h")))
    return any(os.path.getmtime(d) > t for d in deps)


def _run(cmd, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed:\n{res.stdout}\n{res.stderr}")


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compile csrc/*.hip -> sam3_lora_amd/libsam3_lora_amd.so for gfx950."""
    if not force and not needs_build():
        return LIB_PATH
    hipcc = _hipcc()
    with tempfile.TemporaryDirectory(prefix="sam3_lora_amd_build_") as tmp:
        objs = [os.path.join(tmp, os.path.basename(src) + ".o") for src in SRCS]
        cmds = [[hipcc] + FLAGS + ["-I", INCLUDE, "-c", src, "-o", obj] for src, obj in zip(SRCS, objs)]
        with ThreadPoolExecutor(max_workers=min(len(cmds), os.cpu_count() or 1, 8)) as pool:      # one compiler process per unit
            list(pool.map(lambda cmd: _run(cmd, verbose), cmds))
        _run([hipcc, "--offload-arch=gfx950", "-fPIC", "-shared"] + objs + ["-o", LIB_PATH + ".tmp"], verbose)
    os.replace(LIB_PATH + ".tmp", LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(force=True, verbose=True))
