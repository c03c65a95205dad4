"""Build libftk.so (the gfx950 HIP kernels + the C ABI of include/ftk.h) and _calls.so (eager calls into it) in-tree.

    python fast-transformer_amd/build.py

Compiles every csrc/*.hip for gfx950 with hipcc and links them into
fast-transformer_amd/kernels/libftk.so, which the `kernels` package loads, and csrc/ftk_calls.cpp (host code against
torch's headers) into kernels/_calls.so.
"""

import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
INCLUDE = HERE.parent / "include"
OUT = HERE / "kernels" / "libftk.so"
CALLS = HERE / "kernels" / "_calls.so"
OBJ = HERE / "_build"
ARCH = os.environ.get("FTK_OFFLOAD_ARCH", "gfx950")

FLAGS = [
    "-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}",
    # Code objects the torch-bundled HIP runtime (ROCm 7.0) loads.
    "-mcode-object-version=5",
    # No packed FP32 instructions (v_pk_*_f32) anywhere.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function",
    f"-I{INCLUDE}", f"-I{CSRC}",
]


def hipcc():
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(exe).exists():
        raise RuntimeError("hipcc not found: the gfx950 build needs ROCm's hipcc")
    return exe


def _compile(src):
    obj = OBJ / (src.stem + ".o")
    cmd = [hipcc(), *FLAGS, "-c", str(src), "-o", str(obj)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(line for line in proc.stderr.splitlines() if noise not in line)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src.name}:\n{err}")
    return obj, err


def build_calls():
    """Compile csrc/ftk_calls.cpp against torch and link it to libftk.so."""
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    tmp = CALLS.with_suffix(".so.tmp")
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1",
           "-DUSE_ROCM=1", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-isystem{p}" for p in include_paths()], f"-I{sysconfig.get_paths()['include']}", "-isystem/opt/rocm/include",
           str(CSRC / "ftk_calls.cpp"), "-o", str(tmp), *[f"-L{p}" for p in library_paths()], "-lc10", "-lc10_hip",
           "-ltorch_cpu", "-ltorch", "-ltorch_python", f"-L{OUT.parent}", "-l:libftk.so", "-Wl,-rpath,$ORIGIN"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed on ftk_calls.cpp:\n{proc.stderr}")
    os.replace(tmp, CALLS)


def build(verbose=True):
    """Compile all sources and link libftk.so and _calls.so; returns the library's path."""
    OBJ.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(sources))) as pool:
        results = list(pool.map(_compile, sources))
    for obj, err in results:
        if err.strip() and verbose:
            print(err, file=sys.stderr)
    tmp = OUT.with_suffix(".so.tmp")
    cmd = [hipcc(), "-shared", "-fPIC", f"--offload-arch={ARCH}", *[str(o) for o, _ in results], "-o", str(tmp)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stderr}")
    os.replace(tmp, OUT)
    build_calls()
    if verbose:
        print(f"built {OUT} and {CALLS}")
    return OUT


if __name__ == "__main__":
    build()
