"""Build the HIP C-ABI library ``libftx_hip.so`` in-tree for gfx950.

The library links against the HIP runtime that PyTorch ships, so that a
process which imports torch has exactly one HIP runtime and torch streams,
events and allocations are valid handles for the library.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libftx_hip.so"
SOURCES = ("ftx_runtime.hip", "ftx_kernels.hip", "ftx_gemm.hip", "ftx_attention.hip", "ftx_layers.hip",
           "ftx_int8.hip", "ftx_kvcache.hip", "ftx_staged.hip", "ftx_expcode.hip")
OFFLOAD_ARCH = "gfx950"
# The library's serving calls, taking torch tensors (a CPython extension, host code only); it is told which library.
TORCH_SOURCE = CSRC / "ftx_torch.cpp"
TORCH_LIB_PATH = PKG_DIR / "_ftx_torch.so"


def _torch_lib_dir() -> str:
    import torch

    return str(Path(torch.__file__).resolve().parent / "lib")


def hipcc_command(output: Path = LIB_PATH) -> list[str]:
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    torch_lib = _torch_lib_dir()
    return [
        hipcc,
        f"--offload-arch={OFFLOAD_ARCH}",
        "-O3",
        "-std=c++17",
        "-fPIC",
        "-shared",
        "-Wall",
        # Keep the compiler from forming packed-fp32 instructions by itself.
        "-Xclang",
        "-target-feature",
        "-Xclang",
        "-packed-fp32-ops",
        *[str(CSRC / s) for s in SOURCES],
        "-o",
        str(output),
        f"-L{torch_lib}",
        "-lamdhip64",
        f"-Wl,-rpath,{torch_lib}",
        "-Wl,--no-undefined",
    ]


def torch_command(output: Path = TORCH_LIB_PATH) -> list[str]:
    import torch

    include = Path(torch.__file__).resolve().parent / "include"
    torch_lib = _torch_lib_dir()
    return [
        shutil.which("g++") or "/usr/bin/g++",
        "-O2",
        "-std=c++17",
        "-fPIC",
        "-shared",
        "-Wall",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        f"-isystem{include}",
        f"-isystem{include / 'torch/csrc/api/include'}",
        f"-isystem{sysconfig.get_paths()['include']}",
        str(TORCH_SOURCE),
        "-o",
        str(output),
        f"-L{torch_lib}",
        "-ltorch_python",
        "-ltorch",
        "-ltorch_cpu",
        "-lc10",
        "-ldl",
        f"-Wl,-rpath,{torch_lib}",
    ]


def build(verbose: bool = False) -> Path:
    """Compile the library and its torch binding; always rebuilds. Returns the path of the library."""
    _compile(hipcc_command, LIB_PATH, verbose)
    _compile(torch_command, TORCH_LIB_PATH, verbose)
    return LIB_PATH


def _compile(command, path: Path, verbose: bool) -> None:
    tmp = path.with_suffix(".so.tmp")
    cmd = command(tmp)
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True, check=False)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        raise RuntimeError(f"{Path(cmd[0]).name} failed with exit code {proc.returncode}")
    noise = "is not a recognized feature for this target"
    warnings = [ln for ln in (proc.stdout + proc.stderr).splitlines() if ln.strip() and noise not in ln]
    if warnings and verbose:
        sys.stderr.write("\n".join(warnings) + "\n")
    os.replace(tmp, path)


if __name__ == "__main__":
    print(build(verbose=True))
