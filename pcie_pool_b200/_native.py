"""Loader for the native modules ``pcie_pool_b200._C`` and ``pcie_pool_b200._kv``.

On a machine with a visible GPU a missing or broken extension is an error
(raised on first use), never a silent fallback to a slower path.
"""

from __future__ import annotations

import importlib
import os
from types import ModuleType

_MOD: ModuleType | None = None
_KV: ModuleType | None = None
_ERR: BaseException | None = None


def _gpu_visible() -> bool:
    if os.environ.get("CUDA_VISIBLE_DEVICES", None) == "":
        return False
    return any(os.path.exists(p) for p in ("/dev/nvidia0", "/dev/nvidiactl"))


def native(build_if_missing: bool = True) -> ModuleType:
    """Return the loaded extension module, building it in-tree if needed."""
    global _MOD
    if _MOD is None:
        _MOD = _load("pcie_pool_b200._C", build_if_missing)
    return _MOD


def native_kv() -> ModuleType:
    """Return ``pcie_pool_b200._kv``, the paged-KV operators on torch tensors,
    building it in-tree if needed."""
    global _KV
    if _KV is None:
        try:
            import torch  # noqa: F401  (its libraries are the module's)
        except ImportError as exc:
            raise RuntimeError("the paged-KV operators need torch") from exc

        _KV = _load("pcie_pool_b200._kv", True)
    return _KV


def _load(name: str, build_if_missing: bool) -> ModuleType:
    global _ERR
    try:
        return importlib.import_module(name)
    except ImportError as exc:  # pragma: no cover - depends on build state
        _ERR = exc
    if build_if_missing and os.environ.get("PCIE_POOL_NO_BUILD") != "1":
        from . import _build

        _build.build()
        return importlib.import_module(name)
    raise RuntimeError(
        "pcie_pool_b200 native extension is not built; run "
        "`python -m pcie_pool_b200._build`"
        + (" (a GPU is visible, so no fallback is used)" if _gpu_visible() else "")
        + f": {_ERR}"
    ) from _ERR


def available() -> bool:
    try:
        native(build_if_missing=False)
        return True
    except Exception:
        return False
