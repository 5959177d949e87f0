"""A library that is older than the package says so when it is loaded."""

from __future__ import annotations

import shutil
import subprocess

import pytest

from tensorsmith_hip import _lib

pytestmark = pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc unavailable")


def _library(tmp_path, version, names=()):
    source, lib = tmp_path / "old.c", tmp_path / "libold.so"
    source.write_text(f"int tsattn_abi_version(void) {{ return {version}; }}\n"
                      + "".join(f"int {name}(void) {{ return 0; }}\n" for name in names))
    subprocess.run(["gcc", "-shared", "-fPIC", str(source), "-o", str(lib)], check=True)
    return lib


@pytest.mark.parametrize("change", [-1, 1])
def test_another_version_is_refused_before_its_entry_points(change, tmp_path):
    version = _lib.ABI_VERSION + change
    with pytest.raises(RuntimeError, match=f"ABI {version} != expected {_lib.ABI_VERSION}; rebuild"):
        _lib.load(_library(tmp_path, version))


def test_a_library_without_the_paged_cache_asks_for_a_build(tmp_path):
    names = [n for n in _lib.SIGNATURES if "pages4" not in n and n != "tsattn_abi_version"]
    with pytest.raises(RuntimeError, match="built before tsattn_pages4_.*; rebuild"):
        _lib.load(_library(tmp_path, _lib.ABI_VERSION, names))
