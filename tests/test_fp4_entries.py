"""The C entry points of the four-bit operators, without a GPU: every one is declared, and what they refuse or answer before a launch."""
import ctypes
import inspect
import re

import pytest

from glassbox_amd import build, ops


def test_every_entry_point_is_declared():
    used = set(re.findall(r"\.(gb_fp4_\w+)", inspect.getsource(ops)))
    declared = {name for lib in ("fp4_cache", "fp4_attention", "fp4_gemm") for name in ops._SIGS[lib]}
    assert used and used <= declared, used - declared
