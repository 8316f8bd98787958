"""Builds ``libsparsefold_hip.so`` from ``csrc/*.hip`` for gfx950 with hipcc, and from ``csrc/front.cpp`` the host module
through which the serving-step calls reach it from Python.

Objects are compiled in parallel into ``sparsefold_amd/_build/`` and linked in-tree, so the
library travels with the source tree.  Every HIP translation unit is compiled with the
packed-fp32 feature disabled and with MFMA accumulators in VGPRs.
"""
from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sysconfig
from pathlib import Path

from sparsefold_amd._lib import front_path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libsparsefold_hip.so"
INCLUDE = PKG.parent / "include"

ARCH = "gfx950"
HIP_FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-ffp-contract=fast",
    # MFMA accumulators in VGPRs: left to its heuristics the compiler put the attention
    # kernels' accumulators in AGPRs and copied them to VGPRs and back around every tile
    "-mllvm", "-amdgpu-mfma-vgpr-form",
]


def hipcc() -> str:
  for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
    if cand and Path(cand).exists():
      return cand
  raise RuntimeError("hipcc not found; the HIP library cannot be built")


def _compile(src: Path) -> Path:
  obj = BUILD / (src.stem + ".o")
  cmd = [hipcc(), *HIP_FLAGS, f"-I{INCLUDE}", "-c", str(src), "-o", str(obj)]
  res = subprocess.run(cmd, capture_output=True, text=True)
  if res.returncode != 0:
    raise RuntimeError(f"hipcc failed for {src.name}:\n{res.stderr}")
  return obj


def _front_includes() -> list[Path] | None:
  """Where the host module's headers are (torch's for HIP, Python's, HIP's), or None where one kind is not installed."""
  try:
    import torch
  except ImportError:
    return None
  at = Path(torch.__file__).resolve().parent / "include"
  python = Path(sysconfig.get_paths()["include"])
  if not (at / "c10/hip/HIPStream.h").exists() or not (python / "Python.h").exists():
    return None
  return [at, at / "torch/csrc/api/include", python, Path(hipcc()).resolve().parents[1] / "include"]


def _build_front() -> Path | None:
  """The host module, for this Python and the torch that is installed (its name holds their versions); None where its headers are not."""
  includes = _front_includes()
  if includes is None:
    return None
  import torch
  path = front_path()
  tmp = path.with_suffix(".so.tmp")
  cmd = [hipcc(), "-x", "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
         f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}", *(f"-isystem{i}" for i in includes),
         str(CSRC / "front.cpp"), "-o", str(tmp), f"-L{includes[0].parent / 'lib'}", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python"]
  res = subprocess.run(cmd, capture_output=True, text=True)
  if res.returncode != 0:
    raise RuntimeError(f"hipcc failed for front.cpp:\n{res.stderr}")
  os.replace(tmp, path)
  return path


def build(verbose: bool = False) -> Path:
  """Compiles every ``csrc/*.hip`` and links ``libsparsefold_hip.so``, and builds the host module; returns the library's path.

  The library needs neither torch nor Python: it is linked whatever becomes of the host module.  Without the headers of both there is no
  host module (its calls then go through ctypes); one that does not compile is an error."""
  BUILD.mkdir(exist_ok=True)
  srcs = sorted(CSRC.glob("*.hip"))
  with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as ex:
    front = ex.submit(_build_front)
    objs = list(ex.map(_compile, srcs))
  tmp = LIB.with_suffix(".so.tmp")
  cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)]
  res = subprocess.run(cmd, capture_output=True, text=True)
  if res.returncode != 0:
    raise RuntimeError(f"link failed:\n{res.stderr}")
  os.replace(tmp, LIB)
  if verbose:
    print(f"built {LIB}")
  if front.result() is None:
    for stale in LIB.parent.glob("_front-*.so"):               # (of an earlier build, perhaps for another library)
      stale.unlink()
    if verbose:
      print("no host module: torch's or Python's C++ headers are not installed")
  return LIB


if __name__ == "__main__":
  build(verbose=True)
