"""Builds libaspire_b200.so in-tree with nvcc for sm_100a, and _torch_binding.so
(the feed-forward operators' Python calls) with the host compiler.

Usage: ``python -m aspire_b200.build [--verbose-ptxas]``.  Both are written next
to this file so that they travel with the source tree.
"""

from __future__ import annotations

import argparse
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
INCLUDE = PKG_DIR.parent / "include"
LIB_NAME = "libaspire_b200.so"
LIB_PATH = PKG_DIR / LIB_NAME
BINDING_PATH = PKG_DIR / "_torch_binding.so"
BINDING_SOURCE = CSRC / "torch_binding.cpp"

SOURCES = [
    "capi.cu",
    "planner.cpp",
    "attn_gather.cu",
    "attn_tc.cu",
    "attn_merge.cu",
    "append_kv.cu",
    "select_pages.cu",
    "unified_indices.cu",
    "qkv_prologue.cu",
    "plan_device.cu",
    "noalloc.cu",
    "draft_spill.cu",
    "dump_state.cu",
    "capi_ffn.cu",
    "w4_small.cu",
    "w4_tc.cu",
    "moe_route.cu",
    "moe_permute.cu",
    "capi_tree.cu",
    "step_tables.cu",
    "logits.cu",
    "tree_accept.cu",
]

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    cand = shutil.which("nvcc")
    if cand:
        return cand
    default = "/usr/local/cuda/bin/nvcc"
    if os.path.exists(default):
        return default
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libaspire_b200")


def _inputs() -> list[Path]:
    files = [CSRC / s for s in SOURCES]
    files += sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [INCLUDE / "aspire_b200.h"]
    return files


def _older(path: Path, inputs: list[Path]) -> bool:
    if not path.exists():
        return True
    mtime = path.stat().st_mtime
    return any(f.exists() and f.stat().st_mtime > mtime for f in inputs)


def binding_wants() -> str:
    """What a binding built now is for: it works with no other torch or Python."""
    import torch

    return f"torch {torch.__version__}, {sys.implementation.cache_tag}"


def binding_has(path: Path | None = None) -> str | None:
    """What the built binding is for, read from the file (a module of another
    Python cannot be asked); None without one."""
    path = path or BINDING_PATH
    if not path.exists():
        return None
    found = re.search(rb"aspire binding for \[([^\]]*)\]", path.read_bytes())
    return found.group(1).decode() if found else None


def _binding_stale() -> bool:
    return _older(BINDING_PATH, [BINDING_SOURCE, INCLUDE / "aspire_b200.h"]) or binding_has() != binding_wants()


def is_stale() -> bool:
    return _older(LIB_PATH, _inputs()) or _binding_stale()


def _build_binding() -> None:
    import torch

    root = Path(torch.__file__).resolve().parent
    nvcc = Path(nvcc_path()).resolve()
    includes = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
                Path(sysconfig.get_paths()["include"]), nvcc.parent.parent / "include"]
    tmp = BINDING_PATH.with_suffix(".so.tmp")
    cmd = [
        os.environ.get("CXX", "g++"),
        "-O2",
        "-std=c++17",
        "-shared",
        "-fPIC",
        "-fvisibility=hidden",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        f'-DASPIRE_BUILT_FOR="{binding_wants()}"',
        "-I",
        str(INCLUDE),
        *[a for i in includes for a in ("-isystem", str(i))],
        "-o",
        str(tmp),
        str(BINDING_SOURCE),
        f"-L{root / 'lib'}",
        *["-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10"],
    ]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("building _torch_binding.so failed:\n" + " ".join(cmd) + "\n" + proc.stdout + proc.stderr)
    os.replace(tmp, BINDING_PATH)


def build(verbose_ptxas: bool = False, force: bool = False) -> Path:
    """Compiles every CUDA/C++ source of the library into one shared object, and
    the binding."""
    if force or _binding_stale():
        _build_binding()
    if not force and not _older(LIB_PATH, _inputs()):
        return LIB_PATH
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [
        nvcc_path(),
        "-O3",
        "-std=c++17",
        *ARCH_FLAGS,
        "-lineinfo",
        "--threads",
        "8",
        "-shared",
        "-Xcompiler",
        "-fPIC,-fvisibility=hidden",
        "--expt-relaxed-constexpr",
        "-I",
        str(INCLUDE),
        "-o",
        str(tmp),
        *[str(CSRC / s) for s in SOURCES],
    ]
    if verbose_ptxas:
        cmd[1:1] = ["-Xptxas", "-v"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(
            "nvcc failed building libaspire_b200.so:\n" + " ".join(cmd) + "\n" + proc.stdout + proc.stderr
        )
    if verbose_ptxas:
        sys.stderr.write(proc.stdout + proc.stderr)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--verbose-ptxas", action="store_true")
    ap.add_argument("--force", action="store_true")
    args = ap.parse_args()
    path = build(verbose_ptxas=args.verbose_ptxas, force=args.force or args.verbose_ptxas)
    print(path)


if __name__ == "__main__":
    main()
