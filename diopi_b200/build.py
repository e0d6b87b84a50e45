"""Builds the shared libraries of the package with nvcc, in-tree.

  diopi_b200/lib/libdiopi_impl.so  the backend: exported DIOPI ops + sm_100a kernels
  diopi_b200/lib/libdiopi_rt.so    the consumer-side test run time (tensor/context handles)
  diopi_b200/lib/_pycall.*.so      the CPython module that makes the calls of the 8-bit cache operators from torch
                                   tensors, for the Python that runs the build; left out where that has no headers

The backend leaves the diopirt accessors (diopiGetTensorData, diopiGetStream, ...)
undefined, as a DIOPI backend does (impl/CMakeLists.txt:45-46 builds one
libdiopi_impl.so that resolves them from its consumer); everything except the
exported C symbols has hidden visibility. Run as ``python -m diopi_b200.build``.
"""
from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

from ._lib import pycall_name

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "lib"
OBJ = ROOT / "build" / "obj"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = [
    "-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-fvisibility=hidden,-Wall,-Wno-unused-function",
    f"-I{ROOT / 'include'}", f"-I{CSRC}",
]

IMPL_SOURCES = [
    "abi/common.cpp",
    "abi/exports.cpp",
    "abi/tp_group.cpp",
    "kernels/dest_index_copy.cu",
    "kernels/token_decode.cu",
    "kernels/token_decode_gqa.cu",
    "kernels/rms_norm.cu",
    "kernels/rms_norm_backward.cu",
    "kernels/rotary.cu",
    "kernels/apply_penalty.cu",
    "kernels/context_attention.cu",
    "kernels/context_attention_sm100.cu",
    "kernels/matmul_allreduce.cu",
    "kernels/block_table.cu",
    "kernels/quantized_copy_kv.cu",
    "kernels/quantized_attention.cu",
]
RT_SOURCES = ["rt/testrt.cpp"]
PY_SOURCES = ["rt/pycall.cpp"]


def _python_include() -> Path | None:
    """The folder with the headers of the running Python, or None."""
    p = Path(sysconfig.get_paths()["include"])
    return p if (p / "Python.h").exists() else None


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build diopi_b200")
    return exe


def _headers_stamp() -> str:
    h = hashlib.sha1()
    for p in sorted(list(CSRC.rglob("*.hpp")) + list(CSRC.rglob("*.cuh")) + list((ROOT / "include").glob("*.h"))):
        h.update(p.read_bytes())
    h.update(" ".join(COMMON + ARCH).encode())
    return h.hexdigest()[:16]


def _compile(src: str, stamp: str, verbose: bool) -> Path:
    s = CSRC / src
    o = OBJ / (src.replace("/", "_") + f".{stamp}.o")
    if o.exists() and o.stat().st_mtime >= s.stat().st_mtime:
        return o
    for old in OBJ.glob(src.replace("/", "_") + ".*.o"):
        old.unlink()
    cmd = [nvcc(), "-x", "cu", *ARCH, *COMMON, "-c", str(s), "-o", str(o)]
    if src in PY_SOURCES:
        cmd.insert(1, f"-I{_python_include()}")
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
    if verbose or r.stderr.strip():
        sys.stderr.write(r.stderr)
    return o


def _link(objs: list[Path], out: Path, extra: list[str]) -> None:
    cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(out), *map(str, objs), *extra]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link of {out.name} failed:\n{r.stdout}\n{r.stderr}")


def _sources_stamp(sources: list[str], more: str = "") -> str:
    h = hashlib.sha1((_headers_stamp() + more).encode())
    for src in sources:
        h.update((CSRC / src).read_bytes())
    return h.hexdigest()


def _current(files: list[Path], stamp_file: Path, stamp: str) -> bool:
    return all(p.exists() for p in files) and stamp_file.exists() and stamp_file.read_text().strip() == stamp


def build(verbose: bool = False, jobs: int | None = None) -> dict[str, Path]:
    """Compiles what is out of date and returns the paths of the libraries.

    lib/build_stamp.txt holds a hash of every source, header and flag the two libraries were built from, and the call module
    has a stamp of its own; when one matches, nothing of it is compiled (file times do not survive a copy of the tree, hashes do)."""
    LIB.mkdir(parents=True, exist_ok=True)
    out = {"impl": LIB / "libdiopi_impl.so", "rt": LIB / "libdiopi_rt.so"}
    py = LIB / pycall_name()
    libs_stamp, py_stamp = LIB / "build_stamp.txt", LIB / (pycall_name() + ".stamp")
    libs_hash = _sources_stamp(IMPL_SOURCES + RT_SOURCES)
    py_hash = _sources_stamp(PY_SOURCES + RT_SOURCES, pycall_name())   # it makes handles through the run time
    libs = verbose or not _current(list(out.values()), libs_stamp, libs_hash)
    module = verbose or not _current([py], py_stamp, py_hash)
    if module and _python_include() is None:
        sys.stderr.write(f"no Python.h in {sysconfig.get_paths()['include']}: {py.name} is not built\n")
        py.unlink(missing_ok=True)
        module = False
    if libs or module:
        OBJ.mkdir(parents=True, exist_ok=True)
    jobs = jobs or min(8, os.cpu_count() or 1)
    with ThreadPoolExecutor(jobs) as ex:
        def compiled(sources, stamp):
            return list(ex.map(lambda s: _compile(s, stamp, verbose), sources))
        if libs:
            stamp = _headers_stamp()
            impl_objs, rt_objs = compiled(IMPL_SOURCES, stamp), compiled(RT_SOURCES, stamp)
            _link(impl_objs, out["impl"], [])
            _link(rt_objs, out["rt"], [])
            libs_stamp.write_text(libs_hash + "\n")
        if module:
            _link(compiled(PY_SOURCES, py_hash[:16]), py, [])
            py_stamp.write_text(py_hash + "\n")
    return {**out, "py": py} if py.exists() else out


if __name__ == "__main__":
    paths = build(verbose="-v" in sys.argv)
    for k, v in paths.items():
        print(f"{k}: {v}")
