"""The example layer runs: its training loss falls, and generation from the 4-bit cache stays near the layer's own
output on the whole sequence."""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from tattn import _lib
from tests.built import ROOT, ensure_built

ensure_built()


@pytest.mark.gpu
def test_window_layer() -> None:
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    spec = importlib.util.spec_from_file_location("window_layer", os.path.join(ROOT, "examples", "window_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)  # type: ignore[union-attr]
    losses, off = mod.main()
    assert losses[-1] < 0.9 * losses[0]
    # A key or value is off by at most half a code, 1/30 of its group's range: about 0.05 of a normal value's
    # size in the root mean square, and so is a weighted mean of values; scores add as much again.
    assert off < 0.2
    assert _lib.device_status() == 0
