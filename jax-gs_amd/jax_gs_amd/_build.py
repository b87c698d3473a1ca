"""In-tree build of libgsraster.so for gfx950 (hipcc) and of _tensors.so, the host's look at lists
of tensors (g++ against torch's headers); no torch extension machinery."""
from __future__ import annotations

import glob
import os
import subprocess
import sysconfig

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(_HERE), "csrc")
OUT = os.path.join(_HERE, "libgsraster.so")
TENSORS = os.path.join(_HERE, "_tensors.so")

HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    # per-Gaussian arithmetic must round like its sequential float32 statement
    "-ffp-contract=off",
    # float atomicAdd -> hardware global/LDS atomics instead of CAS loops
    "-munsafe-fp-atomics",
    # no packed FP32 instructions (v_pk_*_f32) in generated code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def build_library(verbose: bool = False) -> str:
    """Compile every csrc/*.hip into libgsraster.so (always recompiles)."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    tmp = OUT + ".tmp"
    cmd = [hipcc, *HIPCC_FLAGS, *sources(), "-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, OUT)
    return OUT


def build_tensors(verbose: bool = False) -> str:
    """Compile csrc/gs_tensors.cpp into the module _tensors (always recompiles)."""
    import torch
    from torch.utils import cpp_extension

    tmp = TENSORS + ".tmp"
    include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *[f"-I{i}" for i in include],
           os.path.join(CSRC, "gs_tensors.cpp"), f"-L{cpp_extension.TORCH_LIB_PATH}", "-ltorch_python", "-ltorch",
           "-ltorch_cpu", "-lc10", "-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, TENSORS)
    return TENSORS
