"""Loading the kernel library: one that lacks an entry point serves the others."""
import subprocess
import shutil

import pytest

from axonml_b200 import _native as N


@pytest.fixture
def old_library(tmp_path, monkeypatch):
    """A library from before the int8 operators."""
    src, so = tmp_path / "old.c", tmp_path / "libaxonml_cuda.so"
    src.write_text("int ax_version(void) { return 1; }\n")
    subprocess.run([shutil.which("gcc") or "cc", "-shared", "-fPIC", "-o", str(so), str(src)], check=True)
    monkeypatch.setattr(N, "_LIBDIR", tmp_path)
    monkeypatch.setattr(N, "_CUDA", None)
    monkeypatch.setattr(N, "_ENTRIES", {})
    monkeypatch.delenv("AXONML_BOUNDS", raising=False)
    monkeypatch.delenv("AXONML_REBUILD", raising=False)


def test_an_older_library_keeps_its_entry_points(old_library):
    assert N.cuda().ax_version() == 1


def test_a_missing_entry_point_is_named(old_library):
    with pytest.raises(N.NativeError, match="ax_int8_rows"):
        N.launch("ax_int8_rows", 0)


def test_every_declared_entry_point_is_in_the_built_library():
    lib = N.cuda()._lib
    for name, sig in N._SIGNATURES.items():
        assert len(getattr(lib, name).argtypes) == len(sig)
