"""Build libmi355_tileops.so (HIP kernels + C ABI) for gfx950 with hipcc, in-tree.

``python -m tileops_amd.build`` compiles every translation unit under ``tileops_amd/csrc`` and links
``tileops_amd/lib/libmi355_tileops.so``.  hipcc cross-compiles, so no GPU is needed to build.  Beside it goes
``tileops_amd/lib/_hostcall.so``, the host side of the serving-step calls (a Python module on torch's C++ interface, no device code).
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "lib"
LIB_PATH = LIB_DIR / "libmi355_tileops.so"
HOSTCALL_PATH = LIB_DIR / "_hostcall.so"
OBJ_DIR = PKG / "build"

SOURCES = ["abi.hip", "paged_decode_generic.hip", "paged_decode_mfma.hip", "paged_cache_utils.hip", "paged_cache_step.hip",
           "paged_decode_fp4.hip"]

# -packed-fp32-ops: keep the compiler from forming v_pk_*_f32 out of scalar float code.
HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def _hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found; the MI355X library cannot be built")
    return exe


def _compile(src: str, extra: tuple = (), tag: str = "") -> Path:
    obj = OBJ_DIR / (src + tag + ".o")
    cmd = [_hipcc(), *HIPCC_FLAGS, *extra, "-c", str(CSRC / src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{res.stderr}")
    # the host pass does not know the packed-fp32 feature name and says so; anything else is shown
    noise = "is not a recognized feature for this target"
    rest = [ln for ln in res.stderr.splitlines() if ln.strip() and noise not in ln]
    if rest:
        print("\n".join(rest), file=sys.stderr)
    return obj


def build(verbose: bool = True, extra_flags: tuple = (), lib_path: Path = LIB_PATH) -> Path:
    """Compile and link.  ``extra_flags`` / ``lib_path`` let a developer build an instrumented copy beside the product."""
    OBJ_DIR.mkdir(exist_ok=True)
    lib_path.parent.mkdir(exist_ok=True)
    tag = "" if not extra_flags else "." + lib_path.stem
    with ThreadPoolExecutor(max_workers=min(8, len(SOURCES))) as pool:
        objs = list(pool.map(lambda src: _compile(src, tuple(extra_flags), tag), SOURCES))
    tmp = lib_path.with_suffix(".so.tmp")
    cmd = [_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, lib_path)
    if verbose:
        print(f"built {lib_path} ({lib_path.stat().st_size} bytes)")
    return lib_path


def build_hostcall(verbose: bool = True) -> Path:
    """Compile ``csrc/hostcall.cpp`` against torch and the library (built before)."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        raise RuntimeError("no C++ compiler found; the host side of the serving-step calls cannot be built")
    tmp = HOSTCALL_PATH.with_suffix(".so.tmp")
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for path in (*cpp_extension.include_paths(), sysconfig.get_path("include")):
        cmd += ["-isystem", path]
    cmd += [str(CSRC / "hostcall.cpp"), "-o", str(tmp), "-L", str(LIB_DIR), "-lmi355_tileops"]
    for path in cpp_extension.library_paths():
        cmd += ["-L", path]
    cmd += ["-ltorch_python", "-ltorch_hip", "-ltorch_cpu", "-lc10", "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"compiling hostcall.cpp failed:\n{res.stderr}")
    if res.stderr.strip():
        print(res.stderr, file=sys.stderr)
    os.replace(tmp, HOSTCALL_PATH)
    if verbose:
        print(f"built {HOSTCALL_PATH} ({HOSTCALL_PATH.stat().st_size} bytes)")
    return HOSTCALL_PATH


if __name__ == "__main__":
    build()
    build_hostcall()
