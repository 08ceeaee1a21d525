"""Build libpiekv.so (sm_100a) in-tree with nvcc, and _calls.so with the host compiler.

`python pie_b200/build.py` compiles every CUDA translation unit under pie_b200/csrc into
pie_b200/libpiekv.so.  nvcc cross-compiles without a GPU.  Objects are cached under
pie_b200/csrc/build/ and rebuilt when a source or header is newer.  csrc/calls.cpp, the native way from Python to the
short calls of that library, becomes the extension module pie_b200/_calls.so against the installed torch's headers, and is
built again when torch or the interpreter is another one.
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OBJ = CSRC / "build"
LIB = PKG / "libpiekv.so"
CALLS = PKG / "_calls.so"
CALLS_FOR = OBJ / "calls.txt"  # what _calls.so was built for

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted((PKG.parent / "include").glob("*.h"))


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _torch_version() -> str:
    return importlib.metadata.version("torch")


def _calls_for() -> str:
    return f"torch {_torch_version()}, python {sys.version_info[0]}.{sys.version_info[1]}"


def _calls_stale(hdrs: list[Path]) -> bool:
    return _stale(CALLS, [CSRC / "calls.cpp", *hdrs]) or not CALLS_FOR.exists() or CALLS_FOR.read_text() != _calls_for()


def _torch_has_cuda() -> bool:
    return next(_torch_dir().glob("lib/libc10_cuda.*"), None) is not None


def _torch_dir() -> Path:
    return Path(importlib.util.find_spec("torch").submodule_search_locations[0])


def _calls_command() -> list[str]:
    torch = _torch_dir()
    cuda = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
    # the system's g++: exceptions of torch's libraries pass through, so there must be one C++ runtime
    return [shutil.which("g++") or os.environ.get("CXX", "c++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            "-D_GLIBCXX_USE_CXX11_ABI=1", f'-DPIEKV_TORCH_VERSION="{_torch_version()}"', "-I", str(PKG.parent / "include"), "-I", sysconfig.get_paths()["include"],
            *(x for d in (torch / "include", torch / "include/torch/csrc/api/include", cuda / "include") for x in ("-isystem", str(d))),
            str(CSRC / "calls.cpp"), "-o", str(CALLS), "-L", str(torch / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
            "-ltorch_python"]


def build(verbose: bool = False, force: bool = False, ptxas_info: bool = False) -> Path:
    OBJ.mkdir(parents=True, exist_ok=True)
    nvcc = _nvcc()
    hdrs = _headers()
    jobs = []
    objs = []
    for src in sources():
        obj = OBJ / (src.stem + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + hdrs):
            cmd = [nvcc, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
            if ptxas_info:
                cmd[1:1] = ["-Xptxas", "-v"]
            jobs.append(cmd)

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"compiler failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
        if (verbose or ptxas_info) and (r.stderr.strip() or r.stdout.strip()):
            print(r.stdout + r.stderr, flush=True)

    calls = []
    if force or _calls_stale(hdrs):
        if _torch_has_cuda():
            calls = [_calls_command()]
        else:  # nothing can be launched through such a torch; what runs on the host is used through Python
            print("build: torch without CUDA, _calls.so is left out", flush=True)
    with ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs) + len(calls)))) as ex:
        list(ex.map(run, calls + jobs))
    if calls:
        CALLS_FOR.write_text(_calls_for())
    if jobs or force or _stale(LIB, objs):
        run([nvcc, "-shared", "-o", str(LIB), *map(str, objs), "-gencode", "arch=compute_100a,code=sm_100a",
             "-cudart", "static"])
    return LIB


if __name__ == "__main__":
    out = build(verbose=True, force="--force" in sys.argv, ptxas_info="--ptxas" in sys.argv)
    print(out)
