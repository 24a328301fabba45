"""Build of the CUDA library libbfft.so (nvcc, sm_100a, in-tree).

``build()`` compiles ``csrc/*.cu`` into ``bfft/_lib/libbfft.so`` with
``-gencode arch=compute_100a,code=sm_100a`` and records the compiler version
in ``bfft/_lib/build_meta.json`` (part of the environment fingerprint).  The
library is linked against the static CUDA runtime and carries no torch
dependency; the Python layer loads it with ctypes.  ``csrc/bfft_torch.cpp``
(host code only) becomes the extension module ``bfft/_lib/bfft_torch.so``, which
takes torch tensors to the library's position and cache calls.
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
    return sources() + [TORCH_SRC] + sorted(glob.glob(os.path.join(CSRC, "*.cuh"))) + \
        sorted(glob.glob(os.path.join(INCLUDE, "*.h")))


def source_hash() -> str:
    h = hashlib.sha256()
    for p in _deps():
        with open(p, "rb") as f:
            h.update(os.path.basename(p).encode())
            h.update(f.read())
    return h.hexdigest()[:16]


def build_meta() -> dict | None:
    try:
        with open(META_PATH) as f:
            return json.load(f)
    except (OSError, json.JSONDecodeError):
        return None


def up_to_date() -> bool:
    meta = build_meta()
    return os.path.exists(LIB_PATH) and os.path.exists(TORCH_LIB_PATH) and meta is not None and meta.get("source_hash") == source_hash()


def build_torch_module(verbose: bool = True) -> str:
    """Compile the torch binding against the installed torch's headers, with the
    host compiler that nvcc uses: its C++ runtime has to be torch's own."""
    import sysconfig

    import torch

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
    return TORCH_LIB_PATH


def build(force: bool = False, verbose: bool = True) -> str:
    """Compile libbfft.so and the torch binding if their sources changed; returns the library path."""
    if not force and up_to_date():
        return LIB_PATH
    nvcc = nvcc_path()
    os.makedirs(LIB_DIR, exist_ok=True)
    tmp = LIB_PATH + ".tmp"
    cmd = [nvcc, *ARCH_FLAGS, *NVCC_FLAGS, "-I", INCLUDE, "-o", tmp, *sources()]
    if verbose:
        print("[bfft] " + " ".join(cmd), file=sys.stderr, flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB_PATH)
    build_torch_module(verbose)
    ver = subprocess.run([nvcc, "--version"], capture_output=True, text=True).stdout
    m = re.search(r"release ([0-9.]+), V([0-9.]+)", ver)
    meta = {"nvcc": m.group(2) if m else ver.strip().splitlines()[-1],
            "arch": "sm_100a", "flags": ARCH_FLAGS + NVCC_FLAGS, "source_hash": source_hash()}
    with open(META_PATH, "w") as f:
        json.dump(meta, f, indent=1)
    return LIB_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv)
