"""CPU: what the binding says of a library that was built before entry points were added."""
import subprocess

import pytest

from ufvideo_amd import _lib


@pytest.mark.parametrize("has", [0, 3])
def test_a_library_without_an_entry_point_says_rebuild(tmp_path, monkeypatch, has):
    """same ABI version, but an older build: entries are added without a new version, so the missing name itself is reported, with what to do"""
    src, so = tmp_path / "old.c", tmp_path / "libold.so"
    names = list(_lib.SIGNATURES)[:has]
    src.write_text("int ufv_abi_version(void) { return %d; }\nconst char* ufv_last_error(void) { return \"\"; }\n" % _lib.ABI_VERSION + "".join(f"int {n}(void) {{ return 0; }}\n" for n in names))
    subprocess.run(["gcc", "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    monkeypatch.setattr(_lib, "LIB_PATH", str(so))
    monkeypatch.setattr(_lib, "_lib", None)
    with pytest.raises(_lib.UfvError, match=rf"libold\.so.*{list(_lib.SIGNATURES)[has]}.*rebuild \(make\)"):
        _lib.load()
    assert _lib._lib is None
