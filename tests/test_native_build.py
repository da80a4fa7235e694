"""The in-tree build of the two native modules, with the compiler replaced: the core needs neither torch nor that the
paged-KV operators can be built."""

from pathlib import Path

import pytest

from pcie_pool_b200 import _build

KV = _build.KV_CU_SOURCES + _build.KV_CC_SOURCES


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """What would be run; nothing is, and nothing in the tree is touched."""
    ran = []
    monkeypatch.setattr(_build, "_compile", ran.append)
    monkeypatch.setattr(_build, "BUILD_DIR", tmp_path)
    monkeypatch.setattr(_build, "extension_path", lambda name="_C": tmp_path / f"{name}.so")
    return ran


def made(commands):
    """Names of the sources compiled and of the modules linked."""
    at = [c[c.index("-o") + 1] for c in commands]
    return ({Path(c[c.index("-c") + 1]).name for c in commands if "-c" in c}, [Path(p).name for p in at if p.endswith(".so")])


def test_both_modules_are_built(commands):
    _build.build()
    compiled, linked = made(commands)
    assert compiled == {*_build.CU_SOURCES, *_build.CC_SOURCES, *KV} and linked == ["_C.so", "_kv.so"]


def test_the_core_is_built_where_torch_is_not_installed(commands, monkeypatch, capsys):
    monkeypatch.setattr("importlib.util.find_spec", lambda name: None)
    assert _build.build().name == "_C.so"
    compiled, linked = made(commands)
    assert compiled == {*_build.CU_SOURCES, *_build.CC_SOURCES} and linked == ["_C.so"]
    assert "torch is not installed" in capsys.readouterr().out


def test_the_core_is_linked_before_the_operators_fail(commands, monkeypatch):
    def run(cmd):
        if "-c" in cmd and Path(cmd[cmd.index("-c") + 1]).name in KV:
            raise RuntimeError("native build failed")
        commands.append(cmd)

    monkeypatch.setattr(_build, "_compile", run)
    with pytest.raises(RuntimeError, match="native build failed"):
        _build.build()
    assert made(commands)[1] == ["_C.so"]


def run(code):
    import os
    import subprocess
    import sys

    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                          cwd=Path(__file__).resolve().parents[1], env={**os.environ, "PCIE_POOL_NO_BUILD": "1"})


def test_a_module_of_another_torch_version_is_not_loaded():
    r = run("import importlib.metadata as m\nm.version = lambda name: '1.0'\nfrom pcie_pool_b200._native import native_kv\nnative_kv()")
    assert r.returncode != 0 and "was built for torch" in r.stderr and "this is torch 1.0" in r.stderr


def test_the_operators_name_what_they_need_where_torch_is_missing():
    r = run("import sys\nsys.modules['torch'] = None\nfrom pcie_pool_b200._native import native, native_kv\nnative()\nnative_kv()")
    assert r.returncode != 0 and "RuntimeError: the paged-KV operators need torch" in r.stderr
