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


def test_rotation_tables_are_exact() -> None:
    """The layer as the example makes it has cos and sin to float32's last place: the angles, up to 8191, need more
    bits than float32, and the tables more than the layers' 16. (Without a GPU.)"""
    spec = importlib.util.spec_from_file_location("window_layer", os.path.join(ROOT, "examples", "window_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)  # type: ignore[union-attr]
    layer = mod.make_layer(256, "cpu")
    angle = torch.arange(8192, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, 64, 2).double() / 64)
    assert layer.cos.dtype == layer.sin.dtype == torch.float32
    assert float((layer.cos.double() - angle.cos()).abs().max()) <= 2.0**-24
    assert float((layer.sin.double() - angle.sin()).abs().max()) <= 2.0**-24
    assert layer.qkv.weight.dtype == layer.out.weight.dtype == torch.float16
    assert layer.q_norm.dtype == layer.k_norm.dtype == torch.float32
