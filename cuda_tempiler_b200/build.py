"""Build the in-tree sm_100a shared library ``libtempo_sm100.so`` with nvcc.

The library compiles the SHIPPED artifacts: csrc/tempo_sm100.cu (the C-ABI shim) includes the
launch.cu of kernels/shipped/gemm_fp16/sm_100a and of kernels/shipped/gemm_w8a16/sm_100a, each
of which brings its POD ABI (launch.cuh), the frozen kernels (kernel.cuh) and its generated
dispatch body (dispatch.inc) -- the reference's launch.cu + dispatch.inc scheme.

The library is the product: the CUDA kernels plus the extern "C" entry points declared in
``include/tempo_sm100.h``.  It is built in-tree so that it travels with the repository to the
GPU box; there is no JIT cache and no CPU fallback.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import tempfile
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
SHIPPED = PKG / "kernels" / "shipped"
SKELETON = PKG / "tempo" / "plugins" / "sm100" / "skeletons" / "gemm_sm100"
LIB = PKG / "libtempo_sm100.so"
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put CUDA's bin on PATH)")


def sources() -> list:
    return (sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h"))
            + sorted(SKELETON.glob("*.cuh"))
            + sorted(SHIPPED.glob("*/sm_100a/*.cuh")) + sorted(SHIPPED.glob("*/sm_100a/*.cu"))
            + sorted(SHIPPED.glob("*/sm_100a/*.inc")) + [INCLUDE / "tempo_sm100.h"])


def stale() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    return any(p.stat().st_mtime > t for p in sources())


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every .cu under csrc/ into one shared library (no-op when up to date)."""
    if not force and not stale():
        return LIB
    flags = [*ARCH_FLAGS, "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC"]
    with tempfile.TemporaryDirectory(dir=PKG, prefix="_build") as tmp:
        # the translation units side by side, then one shared library
        jobs = []
        for src in sorted(CSRC.glob("*.cu")):
            obj = os.path.join(tmp, src.stem + ".o")
            cmd = [nvcc(), *flags, "-Xptxas", "-v", f"-I{INCLUDE}", f"-I{CSRC}", f"-I{SHIPPED}",
                   "-c", "-o", obj, str(src)]
            jobs.append((obj, subprocess.Popen(cmd, stdout=subprocess.PIPE,
                                               stderr=subprocess.PIPE, text=True)))
        done = [(obj, p, *p.communicate()) for obj, p in jobs]
        for _, p, out, err in done:
            if p.returncode != 0:
                raise RuntimeError("nvcc failed:\n" + out + err)
        res = subprocess.run([nvcc(), *flags, "-shared", "-o", str(LIB) + ".tmp",
                              *[obj for obj, *_ in done]], capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
    os.replace(str(LIB) + ".tmp", LIB)
    log = "".join(err for *_, err in done)
    (PKG / "libtempo_sm100.ptxas.log").write_text(log)
    if verbose:
        print(log)
    return LIB


if __name__ == "__main__":
    build(force=True)
    print(LIB)
