"""Build libfp8gq.so (the C ABI in include/fp8gq.h) in-tree with nvcc for
sm_100a, and the serving operators' Python binding next to it with g++.  Run
``python -m fp8gq._build`` (with ``sglang-triton-fusion_b200`` on sys.path) or
call :func:`build`.  The library depends on no torch; the binding is of one torch
and Python version, which its name tells, and the operators run without it."""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
SRC_DIR = PKG_DIR.parent / "csrc"
REPO_DIR = PKG_DIR.parent.parent
LIB_PATH = PKG_DIR / "libfp8gq.so"
SOURCES = ["fp8gq_api.cu", "serve_api.cu"]
HEADERS = {"fp8gq_api.cu": ["fp8gq_device.cuh", "host_common.h", "tensor_core.cuh", "gemv_row.cuh", "gemm_tm.cuh",
                            "quant_only.cuh", "swiglu_writer.cuh", "chain.cuh", "add_rmsnorm.cuh", "stack.cuh"],
           "serve_api.cu": ["fp8gq_device.cuh", "host_common.h", "tensor_core.cuh", "rope_append.cuh",
                            "paged_decode.cuh", "prompt_attention.cuh", "token_logprobs.cuh"]}
OBJ_DIR = PKG_DIR / "build"
NATIVE_SOURCE = "serve_python.cpp"               # the serving operators' Python binding

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def nvcc_path() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found (set NVCC or put CUDA's bin/ on PATH)")
    return cand


def _inputs(source: str):
    return [SRC_DIR / source, *[SRC_DIR / h for h in HEADERS[source]], REPO_DIR / "include" / "fp8gq.h"]


def _newer_than(target: Path, files) -> bool:
    if not target.exists():
        return False
    t = target.stat().st_mtime
    return all(f.stat().st_mtime <= t for f in files)


def native_path() -> Path:
    """The binding for this torch and Python."""
    import torch
    return PKG_DIR / f"_serve_native-torch{torch.__version__}-py{sys.version_info[0]}.{sys.version_info[1]}.so"


def library_up_to_date() -> bool:
    return _newer_than(LIB_PATH, [f for s in SOURCES for f in _inputs(s)])


def native_up_to_date() -> bool:
    return _newer_than(native_path(), [SRC_DIR / NATIVE_SOURCE, REPO_DIR / "include" / "fp8gq.h"])


def up_to_date() -> bool:
    return library_up_to_date() and native_up_to_date()


def _native_command(target: str):
    """g++ command of the binding, which links torch's libraries (loaded by then)
    and libfp8gq.so next to it."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths
    inc = [*include_paths(), sysconfig.get_paths()["include"], str(REPO_DIR / "include"),
           str(Path(nvcc_path()).resolve().parent.parent / "include")]
    return [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{i}" for i in inc],
            str(SRC_DIR / NATIVE_SOURCE), "-o", target, f"-L{PKG_DIR}", "-l:libfp8gq.so",
            f"-L{Path(torch.__file__).parent / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
            "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose: bool = False, extra_flags=None) -> Path:
    """Compile libfp8gq.so and the binding, whatever is not already current."""
    build_library(force, verbose, extra_flags)
    build_native(force)
    return LIB_PATH


def build_native(force: bool = False) -> Path:
    """Compile the binding next to this file unless it is already current."""
    path = native_path()
    if force or not native_up_to_date():
        tmp = f"{path}.{os.getpid()}.tmp"
        res = subprocess.run(_native_command(tmp), capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"g++ failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, path)
    return path


def build_library(force: bool = False, verbose: bool = False, extra_flags=None) -> Path:
    """Compile libfp8gq.so next to this file unless it is already current: one
    object per translation unit, in parallel, those that are current reused."""
    if not force and library_up_to_date():
        return LIB_PATH
    OBJ_DIR.mkdir(exist_ok=True)
    jobs = []
    for s in SOURCES:
        obj = OBJ_DIR / (Path(s).stem + ".o")
        if force or extra_flags or not _newer_than(obj, _inputs(s)):
            cmd = [nvcc_path(), *NVCC_FLAGS, *(extra_flags or []), "-I", str(REPO_DIR / "include"),
                   "-c", "-o", str(obj) + ".tmp", str(SRC_DIR / s)]
            if verbose:
                print(" ".join(cmd), file=sys.stderr)
            jobs.append((obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    said = [(obj, p.communicate()[0], p.returncode) for obj, p in jobs]
    for obj, text, rc in said:
        if rc != 0:
            raise RuntimeError(f"nvcc failed ({rc}):\n{text}")
        if verbose and text:
            print(text, file=sys.stderr)
        os.replace(str(obj) + ".tmp", obj)
    link = [nvcc_path(), *NVCC_FLAGS, "-shared", "-o", str(LIB_PATH) + ".tmp",
            *[str(OBJ_DIR / (Path(s).stem + ".o")) for s in SOURCES]]
    res = subprocess.run(link, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    os.replace(str(LIB_PATH) + ".tmp", LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True,
                extra_flags=["-Xptxas", "-v"] if "--ptxas-v" in sys.argv else None))
