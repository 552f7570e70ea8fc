"""Build libppo_hip.so (all HIP sources under csrc/) for gfx950 with hipcc, in-tree.

Usage: ``python -m tt_rsl_rl_amd.build`` (or ``__graft_entry__.build()``).  Sources are compiled in parallel
to objects under ``csrc/_build/`` and linked into ``tt_rsl_rl_amd/libppo_hip.so``.  Beside it the host compiler builds
``tt_rsl_rl_amd/_tensor_table.so`` (csrc/tensor_table.cpp), the one part that reads torch's objects.
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
BUILD_DIR = CSRC / "_build"
LIB = PKG / "libppo_hip.so"
TABLE = PKG / "_tensor_table.so"
ARCH = os.environ.get("PPO_HIP_ARCH", "gfx950")

# -packed-fp32-ops: hipcc must not form v_pk_{add,mul,fma}_f32 by itself on this target.
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{INCLUDE}",
]
# PPO_HIP_TUNING=1 at build time compiles the tile / split / wave variants and their environment overrides used for
# tuning sweeps; the default library holds only the configurations the tests cover.
if os.environ.get("PPO_HIP_TUNING") == "1":
    HIPCC_FLAGS.append("-DPPO_HIP_TUNING")


def hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(exe).exists():
        raise RuntimeError("hipcc not found: the ROCm toolchain is required to build libppo_hip.so")
    return exe


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.hip"))


def _compile(src: Path) -> Path:
    obj = BUILD_DIR / (src.stem + ".o")
    cmd = [hipcc(), *HIPCC_FLAGS, "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    return obj


def compile_table(cxx: str, out: Path, flags: list[str]) -> None:
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    tmp = out.with_suffix(".so.tmp")
    cmd = [cxx, *flags, "-std=c++17", "-fPIC", "-shared", "-Wall", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-I{p}" for p in include_paths()), f"-I{sysconfig.get_paths()['include']}", str(CSRC / "tensor_table.cpp"), "-o", str(tmp),
           *(f"-L{p}" for p in library_paths()), "-ltorch_python", "-ltorch_cpu", "-lc10"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cxx} failed on tensor_table.cpp:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, out)


def _compile_table() -> None:
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        raise RuntimeError("g++ not found: it builds the module that reads torch's tensors")
    compile_table(cxx, TABLE, ["-O2"])


def build(verbose: bool = True) -> Path:
    """Compile every csrc/*.hip and link libppo_hip.so, and build _tensor_table.so.  Always rebuilds."""
    BUILD_DIR.mkdir(parents=True, exist_ok=True)
    srcs = sources()
    if not srcs:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as pool:
        table = pool.submit(_compile_table)
        objs = list(pool.map(_compile, srcs))
        table.result()
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB} from {len(srcs)} sources for {ARCH}", file=sys.stderr)
    return LIB


if __name__ == "__main__":
    build()
