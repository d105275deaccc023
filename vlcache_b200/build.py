"""Build recipe for the in-tree C-ABI library ``vlcache_b200/libvlcache_b200.so``.

Compiles every CUDA translation unit for sm_100a only (tcgen05/TMA code does not
exist on other architectures) with nvcc, links the host planner, and links the
CUDA runtime statically so the library has no torch dependency.  The driver API
(cuTensorMapEncodeTiled) is reached through cudaGetDriverEntryPoint, so the
library also loads on machines without a GPU (CPU-side tests use the planner).  A small Python extension
(``_binding``, g++ against torch's headers) calls it for the ops whose calls are short; where torch is not installed,
the library is built without it.

Usage: ``python -m vlcache_b200.build [--force] [--verbose]``.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import hashlib
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
INCLUDE = REPO_DIR / "include"
BUILD_DIR = REPO_DIR / "_build" / "vlcache_b200"
LIB_PATH = PKG_DIR / "libvlcache_b200.so"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
CUDA_SOURCES = ["runtime.cu", "kv_ops.cu", "prefill_attn.cu", "decode_attn.cu", "metadata.cu", "gemm.cu", "content_hash.cu",
                "rope_axes.cu", "kv_fp4.cu", "decode_fp4.cu", "pages.cu", "decode_window.cu", "decode_window_wide.cu",
                "step_metadata.cu", "verify.cu"]
CPP_SOURCES = ["plan.cpp"]
BINDING_SOURCE = "binding.cpp"
BINDING_PATH = PKG_DIR / "_binding.so"


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; the vlcache_b200 CUDA library cannot be built")
    return cand


def _sources() -> list[Path]:
    return [CSRC / s for s in CUDA_SOURCES + CPP_SOURCES + [BINDING_SOURCE]]


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


STAMP_PATH = LIB_PATH.with_name(LIB_PATH.name + ".srchash")


def source_hash() -> str:
    """SHA-256 over the bytes of every source, header and this recipe (names included), and the versions of
    Python and torch that the binding is built for (none: no binding): the library is rebuilt exactly when this
    differs from the hash it was built from."""
    h = hashlib.sha256(f"{sys.implementation.cache_tag} {_torch_version()}\0".encode())
    for p in _sources() + _headers() + [Path(__file__)]:
        h.update(p.name.encode())
        h.update(b"\0")
        h.update(p.read_bytes())
        h.update(b"\0")
    return h.hexdigest()


def is_fresh() -> bool:
    """True when the in-tree library exists and was built from the current sources."""
    return (LIB_PATH.exists() and (BINDING_PATH.exists() or not _torch_dir()) and STAMP_PATH.exists()
            and STAMP_PATH.read_text().strip() == source_hash())


def _needs_build() -> bool:
    return not is_fresh()


def _compile(src: Path, verbose: bool) -> Path:
    BUILD_DIR.mkdir(parents=True, exist_ok=True)
    obj = BUILD_DIR / (src.name + ".o")
    cmd = [nvcc_path(), *ARCH_FLAGS, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
           "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(src), "-o", str(obj)]
    if src.suffix == ".cu":
        # Relocatable device code: one library-wide device error word across units.
        cmd[1:1] = ["-rdc=true"] + (["-Xptxas", "-v"] if verbose else [])
    else:
        cmd += ["-x", "c++"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    if verbose and (res.stdout or res.stderr):
        sys.stderr.write(res.stdout + res.stderr)
    return obj


def _torch_dir() -> Path | None:
    """Where torch is installed (None: nowhere), without importing it."""
    spec = importlib.util.find_spec("torch")
    return Path(spec.submodule_search_locations[0]) if spec and spec.submodule_search_locations else None


def _torch_version() -> str:
    if not _torch_dir():
        return "none"
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:   # a tree that was not installed
        return "unnamed"


def _compile_binding(verbose: bool) -> Path:
    torch = _torch_dir()
    obj = BUILD_DIR / (BINDING_SOURCE + ".o")
    BUILD_DIR.mkdir(parents=True, exist_ok=True)
    include = [torch / "include", torch / "include/torch/csrc/api/include", sysconfig.get_paths()["include"],
               Path(nvcc_path()).resolve().parent.parent / "include"]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", "-I", str(INCLUDE),
           *[a for p in include for a in ("-isystem", str(p))], "-c", str(CSRC / BINDING_SOURCE), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for {BINDING_SOURCE}:\n{' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    if verbose and (res.stdout or res.stderr):
        sys.stderr.write(res.stdout + res.stderr)
    return obj


def _link_binding(obj: Path) -> None:
    tmp = BINDING_PATH.with_suffix(".so.tmp")
    cmd = ["g++", "-shared", "-o", str(tmp), str(obj), f"-L{_torch_dir() / 'lib'}", "-ltorch_python", "-ltorch_cpu",
           "-lc10_cuda", "-lc10", f"-L{PKG_DIR}", f"-l:{LIB_PATH.name}", "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link of the binding failed:\n{' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, BINDING_PATH)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile (unless the library was built from exactly these sources) and return the
    path of the shared library."""
    if not force and not _needs_build():
        return LIB_PATH
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        binding = ex.submit(_compile_binding, verbose) if _torch_dir() else None
        objs = list(ex.map(lambda s: _compile(s, verbose), [CSRC / s for s in CUDA_SOURCES + CPP_SOURCES]))
        binding_obj = binding.result() if binding else None
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [nvcc_path(), *ARCH_FLAGS, "-rdc=true", "-shared", "-cudart", "static", "-Xcompiler", "-fPIC",
           "-o", str(tmp), *map(str, objs)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    digest = source_hash()
    os.replace(tmp, LIB_PATH)
    if binding_obj:
        _link_binding(binding_obj)
    STAMP_PATH.write_text(digest + "\n")
    return LIB_PATH


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true", help="print ptxas resource usage")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    main()
