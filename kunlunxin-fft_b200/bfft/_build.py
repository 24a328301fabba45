"""Build of the CUDA library libbfft.so (nvcc, sm_100a, in-tree).

``build()`` compiles ``csrc/*.cu`` into ``bfft/_lib/libbfft.so`` with
``-gencode arch=compute_100a,code=sm_100a`` and records the compiler version
in ``bfft/_lib/build_meta.json`` (part of the environment fingerprint).  The
library is linked against the static CUDA runtime and carries no torch
dependency; the Python layer loads it with ctypes.  ``csrc/bfft_torch.cpp``
(host code only) becomes the extension module ``bfft/_lib/bfft_torch.so``, which
takes torch tensors to the library's position and cache calls.  It has a record of
its own (``torch_meta.json``: its sources, and the torch and Python it was compiled
for); where it cannot be compiled (no host compiler, no torch headers), the library
is complete without it and only those calls are missing.
"""
from __future__ import annotations

import glob
import hashlib
import json
import os
import re
import shutil
import subprocess
import sys
import warnings

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
REPO = os.path.dirname(ROOT)
CSRC = os.path.join(ROOT, "csrc")
INCLUDE = os.path.join(REPO, "include")
LIB_DIR = os.path.join(PKG_DIR, "_lib")
LIB_PATH = os.path.join(LIB_DIR, "libbfft.so")
TORCH_SRC = os.path.join(CSRC, "bfft_torch.cpp")
TORCH_LIB_PATH = os.path.join(LIB_DIR, "bfft_torch.so")
META_PATH = os.path.join(LIB_DIR, "build_meta.json")
TORCH_META_PATH = os.path.join(LIB_DIR, "torch_meta.json")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--threads", "0", "-Xcompiler", "-fPIC", "-shared",
              "-Xcompiler", "-fvisibility=hidden", "-Xcompiler", "-Wall"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put /usr/local/cuda/bin on PATH)")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps() -> list[str]:
    return sources() + sorted(glob.glob(os.path.join(CSRC, "*.cuh"))) + \
        sorted(glob.glob(os.path.join(INCLUDE, "*.h")))


def _hash(paths: list[str]) -> str:
    h = hashlib.sha256()
    for p in paths:
        with open(p, "rb") as f:
            h.update(os.path.basename(p).encode())
            h.update(f.read())
    return h.hexdigest()[:16]


def source_hash() -> str:
    return _hash(_deps())


def _read_meta(path: str) -> dict | None:
    try:
        with open(path) as f:
            return json.load(f)
    except (OSError, json.JSONDecodeError):
        return None


def build_meta() -> dict | None:
    return _read_meta(META_PATH)


def up_to_date() -> bool:
    meta = build_meta()
    return os.path.exists(LIB_PATH) and meta is not None and meta.get("source_hash") == source_hash()


def torch_target() -> dict:
    """What a binding is compiled for: the running torch and Python."""
    import sysconfig

    import torch

    return {"torch": torch.__version__, "cxx11_abi": bool(torch._C._GLIBCXX_USE_CXX11_ABI),
            "python": sysconfig.get_config_var("SOABI")}


def torch_module_fits() -> bool:
    """Whether the built binding, if any, was compiled for the running torch and Python."""
    meta = _read_meta(TORCH_META_PATH)
    return os.path.exists(TORCH_LIB_PATH) and meta is not None and meta.get("target") == torch_target()


def torch_module_up_to_date() -> bool:
    return torch_module_fits() and _read_meta(TORCH_META_PATH)["source_hash"] == _torch_hash()


def _torch_hash() -> str:
    return _hash([TORCH_SRC, os.path.join(INCLUDE, "bfft.h")])


def build_torch_module(verbose: bool = True) -> str:
    """Compile the torch binding against the installed torch's headers, with the
    host compiler that nvcc uses: its C++ runtime has to be torch's own.  Raises where
    that fails; a binding of other sources or another torch is gone by then."""
    import sysconfig

    import torch

    for path in (TORCH_META_PATH, TORCH_LIB_PATH):
        if os.path.exists(path):
            os.remove(path)
    os.makedirs(LIB_DIR, exist_ok=True)
    root = os.path.dirname(torch.__file__)
    include = os.path.join(root, "include")
    tmp = TORCH_LIB_PATH + ".tmp"
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", INCLUDE,
           "-I", sysconfig.get_paths()["include"], "-isystem", include,
           "-isystem", os.path.join(include, "torch", "csrc", "api", "include"),
           "-isystem", os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include"),
           "-o", tmp, TORCH_SRC, "-L", os.path.join(root, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10",
           "-lc10_cuda"]
    if verbose:
        print("[bfft] " + " ".join(cmd), file=sys.stderr, flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, TORCH_LIB_PATH)
    with open(TORCH_META_PATH, "w") as f:
        json.dump({"target": torch_target(), "source_hash": _torch_hash()}, f, indent=1)
    return TORCH_LIB_PATH


def _build_library(verbose: bool) -> None:
    nvcc = nvcc_path()
    os.makedirs(LIB_DIR, exist_ok=True)
    tmp = LIB_PATH + ".tmp"
    cmd = [nvcc, *ARCH_FLAGS, *NVCC_FLAGS, "-I", INCLUDE, "-o", tmp, *sources()]
    if verbose:
        print("[bfft] " + " ".join(cmd), file=sys.stderr, flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB_PATH)
    ver = subprocess.run([nvcc, "--version"], capture_output=True, text=True).stdout
    m = re.search(r"release ([0-9.]+), V([0-9.]+)", ver)
    meta = {"nvcc": m.group(2) if m else ver.strip().splitlines()[-1],
            "arch": "sm_100a", "flags": ARCH_FLAGS + NVCC_FLAGS, "source_hash": source_hash()}
    with open(META_PATH, "w") as f:
        json.dump(meta, f, indent=1)


def build(force: bool = False, verbose: bool = True) -> str:
    """Compile libbfft.so and the torch binding if their sources (or the binding's torch)
    changed; returns the library path.  A binding that cannot be compiled is a warning:
    the position and cache calls then raise, and the transforms are there."""
    if force or not up_to_date():
        _build_library(verbose)
    if force or not torch_module_up_to_date():
        try:
            build_torch_module(verbose)
        except (OSError, RuntimeError, subprocess.CalledProcessError) as e:
            warnings.warn(f"bfft_torch.so was not built, position and cache calls will raise: {e}", stacklevel=2)
    return LIB_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv)
