"""Build the sm_100a shared library in-tree: ``python fast-attnres_b200/build.py``.

``nvcc`` compiles the translation units of ``csrc`` side by side (the read, LayerNorm, embedding
and the vocabulary loss; a unit is compiled again when it or a header it includes is newer than
its object file) and links them into ``attnres/_lib/libattnres_b200.so``; ``g++`` builds the torch
operators over its C ABI (``csrc/torch_ops.cpp``) into ``attnres/_lib/attnres_b200_torch.so``.  nvcc
cross-compiles for sm_100a, so no GPU is needed to build.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

ROOT = Path(__file__).resolve().parent
SOURCES = [ROOT / "csrc" / name for name in ("attnres_b200.cu", "norm.cu", "embedding.cu", "loss.cu")]
HEADERS = sorted((ROOT / "csrc").glob("*.cuh")) + [ROOT.parent / "include" / "attnres_b200.h"]
OUTPUT = ROOT / "attnres" / "_lib" / "libattnres_b200.so"
OPERATORS = ROOT / "csrc" / "torch_ops.cpp"
OPERATORS_OUTPUT = ROOT / "attnres" / "_lib" / "attnres_b200_torch.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(found):
        raise RuntimeError("nvcc not found; the sm_100a library cannot be built")
    return found


def up_to_date() -> bool:
    if not OUTPUT.exists():
        return False
    built = OUTPUT.stat().st_mtime
    return all(path.stat().st_mtime <= built for path in [*SOURCES, *HEADERS, Path(__file__)])


def _includes(path: Path, seen: set[Path]) -> set[Path]:
    """`path` and every project header it includes, directly or not."""
    path = path.resolve()
    if path not in seen and path.exists():
        seen.add(path)
        for name in re.findall(r'#include "([^"]+)"', path.read_text()):
            _includes(path.parent / name, seen)
    return seen


def _compile(source: Path, force: bool) -> tuple[Path, str]:
    """Compile one translation unit; returns its object file and what the compiler said."""
    target = OUTPUT.parent / (source.stem + ".o")
    newest = max(path.stat().st_mtime for path in [*_includes(source, set()), Path(__file__)])
    if not force and target.exists() and newest <= target.stat().st_mtime:
        return target, ""
    # ptxas always reports registers and spills (shown only when asked for): the flag also
    # fixes the order in which it lays the kernels out, so every build of the same sources
    # gives the same binary whether or not the report is printed.
    return target, _run([_nvcc(), *NVCC_FLAGS, "-Xptxas", "-v", "-c", str(source), "-o", str(target)])


def _run(command: list[str]) -> str:
    result = subprocess.run(command, capture_output=True, text=True)
    if result.returncode != 0:
        sys.stderr.write(result.stdout + result.stderr)
        raise RuntimeError(f"{command[0]} failed with exit code {result.returncode}")
    return result.stdout + result.stderr


def _build_operators(force: bool) -> Path:
    """The torch operators over the C ABI: host code only, linked against the kernel library."""
    import torch
    from torch.utils import cpp_extension
    newest = max(path.stat().st_mtime for path in [*_includes(OPERATORS, set()), Path(__file__)])
    if not force and OPERATORS_OUTPUT.exists() and newest <= OPERATORS_OUTPUT.stat().st_mtime:
        return OPERATORS_OUTPUT
    cuda = Path(_nvcc()).resolve().parents[1]
    libraries = cpp_extension.library_paths()
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          *(f"-isystem{path}" for path in [*cpp_extension.include_paths(), cuda / "include"]),
          str(OPERATORS), *(f"-L{path}" for path in [*libraries, OUTPUT.parent]),
          "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", f"-l:{OUTPUT.name}",
          "-Wl,-rpath,$ORIGIN", "-o", str(OPERATORS_OUTPUT)])
    return OPERATORS_OUTPUT


def build(*, force: bool = False, verbose: bool = False) -> Path:
    """Compile the library if any source is newer than it; return its path."""
    if not force and up_to_date():
        _build_operators(force)
        return OUTPUT
    OUTPUT.parent.mkdir(parents=True, exist_ok=True)
    with ThreadPoolExecutor(len(SOURCES)) as pool:
        compiled = list(pool.map(lambda source: _compile(source, force), SOURCES))
    if verbose:
        sys.stderr.write("".join(text for _, text in compiled))
    _run([_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared",
          *(str(target) for target, _ in compiled), "-o", str(OUTPUT)])
    _build_operators(force)
    return OUTPUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
