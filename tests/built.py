"""Builds the library and its PyTorch host side where a test run finds them missing (as a fresh checkout does)."""

from __future__ import annotations

import importlib.util
import os

from tattn import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def ensure_built() -> None:
    ext = os.path.join(os.path.dirname(_lib.LIB_PATH), "_torch_ext.so")
    if os.path.exists(_lib.LIB_PATH) and os.path.exists(ext):
        return
    spec = importlib.util.spec_from_file_location("tattn_build", os.path.join(ROOT, "triton-attn_b200", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)  # type: ignore[union-attr]
    mod.build()
    mod.build_extension()
