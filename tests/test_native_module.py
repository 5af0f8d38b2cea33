"""The module of the paged cache's entry points is needed by these alone."""

from __future__ import annotations

import sys

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
