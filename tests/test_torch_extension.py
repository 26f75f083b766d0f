"""not-gpu: libnif.so alone serves every op but the head losses, whose autograd functions are loaded by their first call."""
import importlib.util
import os

import pytest
import torch

from neuron_interpolation_model_fusion_amd import _lib, ops


def _fresh(monkeypatch, present):
    """The binding imported anew, with nif_torch.so there or not."""
    exists = os.path.exists
    monkeypatch.setattr(os.path, 'exists', lambda p: exists(p) and (present or not str(p).endswith('nif_torch.so')))
    spec = importlib.util.spec_from_file_location('nif_lib_anew', _lib.__file__)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_binding_needs_libnif_only(monkeypatch):
    anew = _fresh(monkeypatch, present=False)
    assert anew.lib.nif_version() == _lib.lib.nif_version()
    with pytest.raises(ImportError, match='nif_torch.so is missing'):
        anew.nif_torch
    monkeypatch.setattr(ops, '_lib', anew)
    monkeypatch.setattr(ops, '_same_device', lambda *a: None)  # the tensors' device is looked at first
    with pytest.raises(ImportError, match='nif_torch.so is missing'):
        ops.top_logits(torch.zeros(2, 3), 1)


def test_the_autograd_functions_are_loaded_once(monkeypatch):
    anew = _fresh(monkeypatch, present=True)
    assert 'nif_torch' not in vars(anew)
    try:
        first = anew.nif_torch
        assert vars(anew)['nif_torch'] is first is anew.nif_torch and callable(first.top_logits)
    finally:
        _lib.nif_torch.set_error(_lib.NifError)  # one shared object a process: its errors are the package's again
    with pytest.raises(AttributeError, match='no attribute'):
        anew.nif_other
