"""A library built from older sources is named as such when it is loaded, whichever of its entries or its number tell."""
import shutil
import subprocess

import pytest

NUMBER = "int omni_moe_abi_version(void) { return %d; }\n"


def _load(tmp_path, monkeypatch, source):
    from omni_infer_amd import _lib
    so = str(tmp_path / f"libstale{len(source)}.so")   # a path that was loaded once gives the same library again
    (tmp_path / "stale.c").write_text(source)
    subprocess.run([shutil.which("gcc"), "-shared", "-fPIC", str(tmp_path / "stale.c"), "-o", so], check=True)
    monkeypatch.setattr(_lib, "LIB_PATH", so)
    monkeypatch.setattr(_lib, "_lib", None)
    try:
        return _lib.lib()
    finally:
        assert _lib._lib is None or _lib._lib._name == so


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("source", ["int nothing;\n", NUMBER % 6, NUMBER % 7], ids=["no number", "older number", "entries missing"])
def test_a_library_of_older_sources(source, tmp_path, monkeypatch):
    from omni_infer_amd import _lib
    with pytest.raises(_lib.OmniMoeError, match="rebuild it") as e:
        _load(tmp_path, monkeypatch, source)
    assert "libstale" in str(e.value)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_the_number_is_read_before_the_entries(tmp_path, monkeypatch):
    from omni_infer_amd import _lib
    with pytest.raises(_lib.OmniMoeError, match="ABI version 6"):
        _load(tmp_path, monkeypatch, NUMBER % 6)
    with pytest.raises(_lib.OmniMoeError, match="omni_moe_last_error"):   # the first entry that is not there
        _load(tmp_path, monkeypatch, NUMBER % _lib.ABI_VERSION + "int more;\n")
