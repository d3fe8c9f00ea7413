"""The torch host module is loaded only if it was built from these sources for the torch that is installed."""
import shutil

import pytest

from nablaengine_b200 import build, capi


class _Rebuilt(Exception):
    pass


@pytest.fixture
def module(tmp_path, monkeypatch):
    """A copy of the built module and its stamp, which load_torch takes for the module; a rebuild is told, not made."""
    build.build_torch()
    at = tmp_path / build.TORCH_LIB.name
    shutil.copy(build.TORCH_LIB, at)
    shutil.copy(build._stamp(build.TORCH_LIB), build._stamp(at))
    (tmp_path / build.LIB.name).symlink_to(build.build())  # (which it looks for beside it)

    def rebuild(force=False):
        raise _Rebuilt

    monkeypatch.setattr(build, "TORCH_LIB", at)
    monkeypatch.setattr(build, "build_torch", rebuild)
    monkeypatch.setattr(capi, "_TORCH", [])
    return at


def test_a_current_module_is_loaded(module):
    assert capi.load_torch(build_if_missing=False).__file__ == str(module)


def _another_torch(module, monkeypatch):
    import torch
    monkeypatch.setattr(torch, "__version__", "1.0.0+other")


def _newer_source(module, monkeypatch):
    source = module.parent / "nb_torch.cpp"
    source.write_text(build.TORCH_DEPS[0].read_text() + "// more\n")
    monkeypatch.setattr(build, "TORCH_DEPS", [source, *build.TORCH_DEPS[1:]])


def _another_stamp(module, monkeypatch):
    build._stamp(module).write_text("another build")


def _no_stamp(module, monkeypatch):
    build._stamp(module).unlink()


def _no_module(module, monkeypatch):
    module.unlink()


@pytest.mark.parametrize("change", [_another_torch, _newer_source, _another_stamp, _no_stamp, _no_module])
def test_any_other_module_is_built_again_or_refused(module, monkeypatch, change):
    change(module, monkeypatch)
    with pytest.raises(RuntimeError, match="nablaengine_b200.build"):
        capi.load_torch(build_if_missing=False)
    with pytest.raises(_Rebuilt):
        capi.load_torch()
    assert not capi._TORCH


def test_preparing_a_device_does_not_need_the_module(monkeypatch):
    """Where the module cannot be loaded, only the calls that need it say so."""
    import torch
    from nablaengine_b200 import torch_ffi

    for kind in (RuntimeError, ImportError, FileNotFoundError):
        def fails(build_if_missing=True):
            raise kind("cannot be built here")

        monkeypatch.setattr(torch_ffi, "_NATIVE", [])
        monkeypatch.setattr(capi, "load_torch", fails)
        torch_ffi._prepare_native()
        with pytest.raises(kind, match="cannot be built here"):
            torch_ffi.layer_norm(torch.zeros(2, 3))
