"""Builds libmpl.so (the C-ABI library of include/mpl.h) for gfx950 with hipcc.

Usage: ``python -m model_amd.build`` (or ``__graft_entry__.build()``).  Each
``csrc/*.hip`` file (hipcc) and host-only ``csrc/*.cpp`` file (g++) is
compiled to an object in ``_build/`` in parallel, then linked into
``model_amd/libmpl.so`` (written atomically).  ``csrc/torch/ops.cpp`` (g++, torch's
headers) becomes the extension module ``model_amd/_ops.so`` beside it.
"""

from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(ROOT, "_build", "obj")
LIB = os.path.join(HERE, "libmpl.so")
OPS = os.path.join(HERE, "_ops.so")
ARCH = "gfx950"

# Packed fp32 VALU ops are disabled for every device compile.  MFMA results
# go to ordinary VGPRs (gfx950's unified register file): the selection code
# reads every score with VALU ops, and accumulators in AGPRs would need a copy
# per element that the scheduler hoists next to the MFMAs, stalling on them.
FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-mllvm", "-amdgpu-mfma-vgpr-form",
    "-Wall", "-Wno-unused-function", "-Wno-unused-variable",
]

# Flags of single files, beyond FLAGS.  score_sort.hip: no IEEE mode and no NaN
# handling of min / max, whose canonicalisation would add an instruction to
# every key (the file turns NaN scores into -FLT_MAX, by integer operations on
# their bits, before they become keys).
FILE_FLAGS = {"score_sort.hip": ["-fno-honor-nans", "-mno-amdgpu-ieee"]}


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (ROCm is required to build libmpl.so)")


# Host-only C++ sources (csrc/*.cpp: no device code) are built with the host
# compiler.
HOST_FLAGS = ["-O3", "-std=c++17", "-fPIC", "-pthread", "-Wall", "-Wno-unused-function"]


def host_cxx() -> str:
    for cand in (os.environ.get("CXX"), shutil.which("g++"), shutil.which("c++")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("no host C++ compiler (g++) found")


def _compile(src: str, cc: str) -> str:
    obj = os.path.join(OBJ, os.path.basename(src) + ".o")
    if src.endswith(".cpp"):
        cmd = [host_cxx(), *HOST_FLAGS, "-c", src, "-o", obj]
    else:
        cmd = [cc, *FLAGS, *FILE_FLAGS.get(os.path.basename(src), []), "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj


def _compile_ops() -> str:
    """The object of csrc/torch/ops.cpp."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    src, obj = os.path.join(CSRC, "torch", "ops.cpp"), os.path.join(OBJ, "torch_ops.o")
    rocm = os.path.dirname(os.path.dirname(hipcc()))
    rocm = rocm if os.path.isdir(os.path.join(rocm, "include", "hip")) else "/opt/rocm"
    inc = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(rocm, "include")]
    cmd = [host_cxx(), "-O2", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function", "-D__HIP_PLATFORM_AMD__=1",
           "-DUSE_ROCM=1", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f for i in inc for f in ("-isystem", i)), "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed for {src}:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj


def _link(cmd, out: str) -> None:
    tmp = out + f".tmp{os.getpid()}"
    r = subprocess.run([*cmd, "-o", tmp], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, out)


def _link_ops(obj: str) -> None:
    from torch.utils import cpp_extension

    libs = [f"-L{p}" for p in cpp_extension.library_paths()]
    _link([host_cxx(), "-shared", "-fPIC", obj, f"-L{HERE}", "-lmpl", *libs, "-ltorch", "-ltorch_cpu", "-ltorch_hip",
           "-lc10", "-lc10_hip", "-ltorch_python", "-Wl,-rpath,$ORIGIN"], OPS)


def build(verbose: bool = False, jobs: int = 8) -> str:
    """Builds both libraries.  libmpl.so needs hipcc and a host compiler alone: it
    is linked first, whatever becomes of the extension module, which needs torch."""
    cc = hipcc()
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")) + glob.glob(os.path.join(CSRC, "*.cpp")))
    with cf.ThreadPoolExecutor(max_workers=max(1, min(jobs, len(srcs) + 1))) as ex:
        ops = ex.submit(_compile_ops)
        objs = list(ex.map(lambda s: _compile(s, cc), srcs))
        _link([cc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-pthread", *objs], LIB)
        try:
            _link_ops(ops.result())
        except Exception as e:
            raise RuntimeError(f"{LIB} is built, {OPS} is not: {e}") from e
    if verbose:
        print(f"built {LIB} from {len(srcs)} sources, and {OPS}")
    return LIB


if __name__ == "__main__":
    build(verbose=True, jobs=int(sys.argv[1]) if len(sys.argv) > 1 else 8)
