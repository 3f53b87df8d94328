"""A library built from other sources is refused with a text that says so,
before its functions are looked up."""

import pytest

from autoindexer_b200 import _lib


class _Fn:
    def __init__(self, value=0):
        self.value = value

    def __call__(self, *args):
        return self.value


class _Library:
    """Has the functions named, and no others."""

    def __init__(self, version, names):
        self.ai_attn_abi_version = _Fn(version)
        for n in names:
            setattr(self, n, _Fn())


@pytest.mark.parametrize("version,names,text", [
    (8, (), "ABI 8"),
    (_lib.ABI_VERSION, (), "rebuild"),
    (_lib.ABI_VERSION, [n for n in _lib.EXPORTED_SYMBOLS if n not in ("ai_attn_abi_version", "ai_verify_draft")], "ai_verify_draft"),
])
def test_other_libraries_are_refused(version, names, text, monkeypatch):
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib.ctypes, "CDLL", lambda path: _Library(version, names))
    with pytest.raises(RuntimeError, match=text) as e:
        _lib.lib()
    assert "rebuild" in str(e.value)
    assert _lib._lib is None


def test_a_library_with_every_function_is_taken(monkeypatch):
    monkeypatch.setattr(_lib, "_lib", None)
    want = _Library(_lib.ABI_VERSION, [n for n in _lib.EXPORTED_SYMBOLS if n != "ai_attn_abi_version"])
    monkeypatch.setattr(_lib.ctypes, "CDLL", lambda path: want)
    assert _lib.lib() is want
