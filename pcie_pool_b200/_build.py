"""In-tree build of the native modules ``pcie_pool_b200._C`` (the core) and
``pcie_pool_b200._kv`` (the paged-KV operators' entry points on torch tensors).

CUDA sources are compiled by nvcc for sm_100a only
(``-gencode arch=compute_100a,code=sm_100a``); host sources by g++.  The CUDA
runtime is linked statically and the driver is reached through
``cudaGetDriverEntryPointByVersion``, so the module builds and imports on a
machine without a GPU.  Objects are cached under ``_build/`` and rebuilt when
their source or any header in ``csrc/`` is newer.

The reference builds its ``_turbobus`` module through CMake without an
architecture list (cpp/CMakeLists.txt:1-45); this build pins the Blackwell
target explicitly.
"""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
BUILD_DIR = PKG_DIR / "_build"
CUDA_HOME = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))

CU_SOURCES = ["ppb_common.cu", "pool_kernels.cu", "engine.cu", "native_ops.cu", "noalloc.cu", "vmm.cu"]
CC_SOURCES = ["planner.cc", "host_ops.cc", "bindings.cc", "bind_ops.cc"]
# the paged-KV operators: a module of its own, since it is built against torch's library
KV_CU_SOURCES = ["kv_attention.cu", "kv_blocks.cu"]
KV_CC_SOURCES = ["torch_kv.cc"]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def extension_path(name: str = "_C") -> Path:
    suffix = sysconfig.get_config_var("EXT_SUFFIX") or ".so"
    return PKG_DIR / f"{name}{suffix}"


def _torch_paths() -> tuple[str, Path] | None:
    """torch's version and folder, without importing it; None where it is not installed."""
    import importlib.metadata
    import importlib.util

    spec = importlib.util.find_spec("torch")
    if spec is None:
        return None
    return importlib.metadata.version("torch"), Path(spec.submodule_search_locations[0])


def _includes() -> list[str]:
    import pybind11

    return [
        f"-I{CSRC}",
        f"-I{pybind11.get_include()}",
        f"-I{sysconfig.get_paths()['include']}",
        f"-I{CUDA_HOME / 'include'}",
    ]


def _newest_header() -> float:
    heads = list(CSRC.glob("*.h")) + list(CSRC.glob("*.cuh"))
    return max((p.stat().st_mtime for p in heads), default=0.0)


def _stale(src: Path, obj: Path, head_mtime: float) -> bool:
    if not obj.exists():
        return True
    m = obj.stat().st_mtime
    return m < src.stat().st_mtime or m < head_mtime


def _compile(cmd: list[str]) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(
            "native build failed:\n" + " ".join(cmd) + "\n" + res.stdout + res.stderr
        )


def build(force: bool = False, verbose: bool = False, jobs: int | None = None) -> Path:
    """Compile (if needed) and link ``_C``, then ``_kv``; returns ``_C``'s path.
    ``_C`` needs neither torch nor that ``_kv`` can be built; without torch ``_kv``
    is left out."""
    BUILD_DIR.mkdir(exist_ok=True)
    nvcc = str(CUDA_HOME / "bin" / "nvcc")
    inc = _includes()
    head = _newest_header()
    torch_paths = _torch_paths()

    def objects(cmds: list, names: list[str], compiler: list[str], includes: list[str], tag: str = "") -> list[Path]:
        """Objects of the sources; what has to be compiled for them joins ``cmds``."""
        objs = []
        for name in names:
            src, obj = CSRC / name, BUILD_DIR / f"{name}{tag}.o"
            objs.append(obj)
            if force or _stale(src, obj, head):
                cmds.append([*compiler, *includes, "-c", str(src), "-o", str(obj)])
        return objs

    cuda = [nvcc, *ARCH_FLAGS, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden"]
    host = ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden"]
    cudart = [f"-L{CUDA_HOME / 'lib64'}", "-lcudart_static", "-lrt", "-lpthread", "-ldl"]
    core_cmds: list[list[str]] = []
    kv_cmds: list[list[str]] = []
    core = objects(core_cmds, CU_SOURCES, cuda, inc) + objects(core_cmds, CC_SOURCES, host, inc)
    if torch_paths:
        version, torch_dir = torch_paths
        torch_inc = [f"-I{CSRC}", f"-isystem{torch_dir / 'include'}", f"-isystem{torch_dir / 'include/torch/csrc/api/include'}",
                     f"-I{sysconfig.get_paths()['include']}", f"-I{CUDA_HOME / 'include'}"]
        kv = objects(kv_cmds, KV_CU_SOURCES, cuda, [f"-I{CSRC}"])
        # its objects are one torch version's
        kv += objects(kv_cmds, KV_CC_SOURCES, [*host, "-DTORCH_EXTENSION_NAME=_kv", f'-DPPB_TORCH="{version}"'], torch_inc, f".torch-{version}")
    with ThreadPoolExecutor(max_workers=jobs or min(8, os.cpu_count() or 4)) as pool:
        core_runs, kv_runs = ([pool.submit(_compile, c) for c in cmds] for cmds in (core_cmds, kv_cmds))
        for run in core_runs:
            run.result()
        out = extension_path()
        if force or core_cmds or not out.exists():
            _compile(["g++", "-shared", "-o", str(out), *map(str, core), *cudart])
        for run in kv_runs:
            run.result()
    if not torch_paths:
        print(f"built {out}; torch is not installed, so the paged-KV operators (_kv) are left out")
        return out
    kv_out, stamp = extension_path("_kv"), BUILD_DIR / "_kv.torch"
    if force or kv_cmds or not kv_out.exists() or not stamp.exists() or stamp.read_text() != version:
        # torch is imported before the module: its libraries are found by their names
        _compile(["g++", "-shared", "-o", str(kv_out), *map(str, kv), f"-L{torch_dir / 'lib'}", "-lc10", "-lc10_cuda",
                  "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python", "-Wl,--exclude-libs,ALL", *cudart])
        stamp.write_text(version)
    if verbose:
        print(f"built {out} and {kv_out}")
    return out


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
