"""CPU checks of what the compiled binding is built for."""

import os

import pytest

from aspire_b200 import _capi, build


def _other(tmp_path, old: bytes, new: bytes):
    """A copy of the built binding, newer than the sources, that claims to be for something else."""
    path = tmp_path / "_torch_binding.so"
    data = build.BINDING_PATH.read_bytes()
    assert data.count(old) >= 1 and len(old) == len(new)
    path.write_bytes(data.replace(old, new))
    return path


def test_the_built_binding_is_for_this_torch_and_python(built_library):
    assert build.binding_has() == build.binding_wants()
    assert not build._binding_stale()
    assert _capi.ops().built_for == f"aspire binding for [{build.binding_wants()}]"


@pytest.mark.parametrize("what", ["torch", "python"])
def test_a_binding_for_another_torch_or_python_is_refused_and_built_again(built_library, monkeypatch, tmp_path, what):
    wants = build.binding_wants().encode()
    part = wants.split(b", ")[0 if what == "torch" else 1]
    path = _other(tmp_path, b"aspire binding for [" + wants, b"aspire binding for [" + wants.replace(part, part[:-1] + b"x"))
    os.utime(path)
    monkeypatch.setattr(build, "BINDING_PATH", path)
    monkeypatch.setattr(_capi, "_ops", None)
    with pytest.raises(RuntimeError, match="python -m aspire_b200.build"):
        _capi.ops()
    assert build.is_stale()
    built = []
    monkeypatch.setattr(build, "_build_binding", lambda: built.append(True))
    build.build()  # what the message asks for
    assert built


def test_a_missing_binding_is_named(built_library, monkeypatch, tmp_path):
    monkeypatch.setattr(build, "BINDING_PATH", tmp_path / "none.so")
    monkeypatch.setattr(_capi, "_ops", None)
    assert build.is_stale()
    with pytest.raises(RuntimeError, match="missing"):
        _capi.ops()
