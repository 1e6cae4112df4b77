"""CPU tests of how the libraries are loaded and built."""
import os
import subprocess

import pytest


def _stub(tmp_path, names):
    src = tmp_path / "stub.c"
    src.write_text("".join("int %s(void) { return 0; }\n" % n for n in names) +
                   'const char *umr_version(void) { return "stub"; }\nconst char *umr_build_id(void) { return "stub"; }\n')
    so = str(tmp_path / "libstub.so")
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-o", so, str(src)])
    return so


def test_an_experimental_build_of_the_render_path_loads(tmp_path, monkeypatch):
    """tools/build_variant.py and tools/exp_pair_cache.py build the render path's sources alone; a missing render symbol still fails"""
    from umr_amd import _lib
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.delenv("UMR_DEBUG_SET", raising=False)
    own = [n for n in _lib.SIGNATURES if n not in ("umr_version", "umr_build_id")]
    monkeypatch.setattr(_lib, "LIB_PATH", _stub(tmp_path, own))
    handle = _lib.lib()
    assert _lib.version() == "stub" and not hasattr(handle, "umr_linear_forward")
    monkeypatch.setattr(_lib, "_lib", None)
    os.makedirs(tmp_path / "b")
    monkeypatch.setattr(_lib, "LIB_PATH", _stub(tmp_path / "b", own[1:]))
    with pytest.raises(AttributeError):
        _lib.lib()
