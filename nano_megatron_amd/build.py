"""Build libnmb.so (the gfx950 kernels behind include/nmb.h) in-tree with hipcc, and
_autograd.so (the autograd nodes in C++ that call it) against the installed torch.

Usage: ``python -m nano_megatron_amd.build`` or ``nano_megatron_amd.build.build()``.
Both land next to this file so they travel with the source tree.
"""

from __future__ import annotations

import concurrent.futures
import os
import pathlib
import shutil
import subprocess
import sys
import sysconfig

import torch

PKG_DIR = pathlib.Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
BUILD_DIR = PKG_DIR / "_build"
LIB_PATH = PKG_DIR / "libnmb.so"
NODES_PATH = PKG_DIR / "_autograd.so"
ROOT = PKG_DIR.parent

ARCH = os.environ.get("NMB_OFFLOAD_ARCH", "gfx950")

HIP_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-fPIC",
    "-std=c++17",
    "-Wall",
    "-Wno-unused-function",
    # packed fp32 VALU ops are disabled for every kernel in this library
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    f"-I{ROOT / 'include'}",
]


def _hipcc() -> str:
    path = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(path):
        raise RuntimeError("hipcc not found; ROCm is required to build libnmb.so")
    return path


def _compile(src: pathlib.Path) -> pathlib.Path:
    obj = BUILD_DIR / (src.stem + ".o")
    cmd = [_hipcc(), *HIP_FLAGS, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    out = "\n".join(
        line
        for line in (proc.stdout + proc.stderr).splitlines()
        if "packed-fp32-ops" not in line  # host pass does not know the device feature
    )
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{out}")
    if out.strip():
        print(out, file=sys.stderr)
    return obj


def _run(cmd: list[str], what: str) -> None:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{proc.stdout}{proc.stderr}")


def _compile_nodes(src: pathlib.Path) -> pathlib.Path:
    """Host code only: g++ against torch's headers."""
    from torch.utils import cpp_extension

    obj = BUILD_DIR / (src.stem + ".o")
    includes = [*cpp_extension.include_paths("cuda"), sysconfig.get_paths()["include"]]
    _run(["g++", "-O2", "-fPIC", "-std=c++17", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f"-DTORCH_EXTENSION_NAME={NODES_PATH.stem}",
          *(f"-isystem{path}" for path in includes), "-c", str(src), "-o", str(obj)], f"g++ of {src.name}")
    return obj


def _link_nodes(obj: pathlib.Path) -> None:
    torch_lib = pathlib.Path(torch.__file__).resolve().parent / "lib"
    tmp = NODES_PATH.with_suffix(".so.tmp")
    _run(["g++", "-shared", str(obj), "-o", str(tmp), f"-L{torch_lib}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch",
          "-ltorch_python", f"-L{PKG_DIR}", f"-l:{LIB_PATH.name}", "-Wl,-rpath,$ORIGIN"], "link of the autograd nodes")
    os.replace(tmp, NODES_PATH)


def build(verbose: bool = True) -> pathlib.Path:
    """Compile every csrc/*.hip for gfx950 and link libnmb.so, then csrc/autograd.cpp and
    _autograd.so; returns the library's path."""
    BUILD_DIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    workers = min(len(sources), max(1, (os.cpu_count() or 2)))
    with concurrent.futures.ThreadPoolExecutor(max_workers=workers) as pool:
        nodes = pool.submit(_compile_nodes, CSRC / "autograd.cpp")
        objs = list(pool.map(_compile, sources))
        nodes_obj = nodes.result()
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [_hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)]
    _run(cmd, "link")
    os.replace(tmp, LIB_PATH)
    _link_nodes(nodes_obj)
    if verbose:
        print(f"built {LIB_PATH} from {len(sources)} sources, and {NODES_PATH.name}", file=sys.stderr)
    return LIB_PATH


if __name__ == "__main__":
    build()
