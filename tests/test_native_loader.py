"""A library that was built from other sources is refused with its name and what to do."""

import ctypes
import subprocess

import pytest

from moe_inference_verify_microbench_b200 import _native


def build(tmp_path, version, functions):
    src = tmp_path / "lib.c"
    src.write_text(f"int moe_abi_version(void) {{ return {version}; }}\n"
                   + "".join(f"int {n}(void) {{ return 0; }}\n" for n in functions))
    lib = tmp_path / "lib.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    return str(lib)


@pytest.fixture
def fresh(monkeypatch):
    monkeypatch.setattr(_native, "_lib", None)


def others():
    return [n for n in _native.SIGNATURES if n != "moe_abi_version"]


def test_library_without_an_entry_point(tmp_path, fresh):
    names = [n for n in others() if n != "moe_w4_layer_forward"]
    path = build(tmp_path, _native.ABI_VERSION, names)
    with pytest.raises(_native.NativeLibraryError, match="moe_w4_layer_forward") as err:
        _native.load(path)
    assert path in str(err.value) and "build" in str(err.value)
    assert _native._lib is None


def test_library_of_another_version(tmp_path, fresh):
    """Told before any missing entry point is."""
    path = build(tmp_path, _native.ABI_VERSION - 1, [])
    with pytest.raises(_native.NativeLibraryError, match="version"):
        _native.load(path)


def test_complete_library(tmp_path, fresh):
    lib = _native.load(build(tmp_path, _native.ABI_VERSION, others()))
    assert lib.moe_abi_version() == _native.ABI_VERSION
    assert isinstance(lib.moe_w4_pack, ctypes._CFuncPtr)
