"""The module of the paged cache's entry points is needed by these alone."""

from __future__ import annotations

import subprocess
import sys
import sysconfig
import types
from pathlib import Path

import pytest
import torch

import turbo_roformer_amd
from turbo_roformer_amd import _hip
from turbo_roformer_amd.paged import HipPagedCache


@pytest.fixture()
def unloaded(monkeypatch):
    """A process that has loaded neither library, on a machine that looks like a gfx950 one."""
    monkeypatch.setattr(_hip, "_lib", None)
    monkeypatch.setattr(_hip, "_native", None)
    monkeypatch.setattr(_hip, "support", lambda: (True, "gfx950"))
    monkeypatch.setattr(torch.cuda, "init", lambda: None)
    return monkeypatch


def _without_module(monkeypatch):
    monkeypatch.delattr(turbo_roformer_amd, "_native", raising=False)
    monkeypatch.setitem(sys.modules, "turbo_roformer_amd._native", None)


def test_the_library_loads_without_it(unloaded):
    _without_module(unloaded)
    assert _hip.load().trf_abi_version() == _hip.ABI_VERSION


def test_the_paged_entry_points_say_that_it_is_missing(unloaded):
    _without_module(unloaded)
    with pytest.raises(_hip.HipUnavailable, match="_native"):
        HipPagedCache(2, 64, device="cpu")
    with pytest.raises(_hip.HipUnavailable, match="_native"):
        _hip.page_release(None, None, None, None, 16, None)


def test_it_is_bound_at_the_first_paged_call(unloaded):
    _hip.load()
    assert _hip._native is None
    HipPagedCache(2, 64, device="cpu")
    assert _hip._native is not None


def test_its_name_carries_the_pythons_tag():
    native = _hip.bind_native(_hip.open_library())
    assert native.__file__.endswith(sysconfig.get_config_var("EXT_SUFFIX"))


@pytest.mark.parametrize("attributes", [{}, dict(abi_version=_hip.ABI_VERSION), dict(abi_version=_hip.ABI_VERSION - 1, functions=("trf_page_plan",) * 4),
                                        dict(abi_version=_hip.ABI_VERSION, functions=("trf_page_plan", "trf_no_such_function"))])
def test_a_module_of_another_library_is_not_bound(monkeypatch, attributes):
    """One that takes functions this library does not have, or has with other arguments."""
    lib = _hip.open_library()
    other = types.ModuleType("turbo_roformer_amd._native")
    other.bind = lambda *addresses: pytest.fail("bound")
    vars(other).update(attributes)
    monkeypatch.setattr(turbo_roformer_amd, "_native", other, raising=False)
    monkeypatch.setitem(sys.modules, "turbo_roformer_amd._native", other)
    monkeypatch.setattr(_hip, "_native", None)
    with pytest.raises(_hip.HipUnavailable, match="not of this library"):
        _hip.bind_native(lib)
    assert _hip._native is None


def test_the_library_builds_without_python():
    """Its makefile's default target names no file of the module."""
    csrc = Path(__file__).resolve().parents[1] / "turbo-roformer_amd" / "csrc"
    plan = subprocess.run(["make", "-n", "-B", "-C", str(csrc), "PYTHON=/no/such/python"], capture_output=True, text=True, check=True)
    assert "libtrf_hip.so" in plan.stdout and "trf_python.cpp" not in plan.stdout


def test_a_tensor_without_an_address_raises(tmp_path):
    """torch.vmap's: in a process of its own, which an exception thrown without the interpreter's lock would end."""
    script = tmp_path / "vmapped.py"
    script.write_text(f"""
import sys
sys.path.insert(0, {str(Path(_hip.__file__).resolve().parents[1])!r})
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from turbo_roformer_amd import _hip
native = _hip.bind_native(_hip.open_library())
with FakeTensorMode():
    ints = lambda *shape: torch.empty(*shape, dtype=torch.int32, device="cuda:0")
    pool, state, table = ints(8), ints(4), ints(2, 4)

    def release(done):
        try:
            native.page_release(0, 0, state, done, pool, table, 16, state)
        except RuntimeError:
            print("raised")
        return done

    torch.vmap(release)(torch.empty(3, 2, dtype=torch.bool, device="cuda:0"))
""")
    run = subprocess.run([sys.executable, str(script)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout == "raised\n", run
