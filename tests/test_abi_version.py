"""A library that is older than the package says so when it is loaded."""

from __future__ import annotations

import shutil
import subprocess

import pytest

from tensorsmith_binding import _tsattn as binding
from tensorsmith_hip import _lib


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc unavailable")
@pytest.mark.parametrize("version", [9, _lib.ABI_VERSION - 1, _lib.ABI_VERSION + 1])
def test_another_version_is_refused_before_its_entry_points(version, tmp_path):
    """Version 9 came without the paged cache's entry points."""
    source, lib = tmp_path / "old.c", tmp_path / "libold.so"
    source.write_text(f"int tsattn_abi_version(void) {{ return {version}; }}\n")
    subprocess.run(["gcc", "-shared", "-fPIC", str(source), "-o", str(lib)], check=True)
    with pytest.raises(RuntimeError, match=f"ABI {version} != expected {_lib.ABI_VERSION}; rebuild"):
        _lib.load(lib)
    with pytest.raises(RuntimeError, match=f"ABI {version}; this binding needs {_lib.ABI_VERSION}"):
        binding.load(str(lib))
