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


def library(name):
    """As built, its entry points declared (``ops`` asks for a GPU before it loads one)"""
    lib = build.load(name)
    for fn, args in ops._SIGS[name].items():
        getattr(lib, fn).argtypes = args
        getattr(lib, fn).restype = ctypes.c_longlong if fn.endswith("_floats") else ctypes.c_int
    lib.gb_last_error.restype = ctypes.c_char_p
    return lib


@pytest.mark.parametrize("hd", [-64, 0, 16, 48, 160, 288, 320, 512, 1 << 20])
def test_heads_that_attention_does_not_take_need_no_workspace(hd):
    """(The model of the launches' times has numbers for the heads that it takes alone.)"""
    floats = library("fp4_attention").gb_fp4_attention_floats
    assert floats(1, 32, 8, 128, 300, 16000, 0, ops.BF16) > 0
    assert floats(1, 32, 8, hd, 300, 16000, 0, ops.BF16) == 0 and floats(1, 32, 8, hd, 1, 16000, 0, ops.F32) == 0


@pytest.mark.parametrize("most", [2 ** 31 - 1, 2 ** 31 - 64, 2 ** 31 - 512])
@pytest.mark.parametrize("hd", [64, 128])
def test_rows_whose_columns_pass_32_bits_are_refused(most, hd):
    """``max_q_len`` says how many rows a launch is laid out for: the numbers of a last workgroup's columns, which begin above the request's, stay
    below 2^31."""
    width = max(64 * r for r in (1, 2, 3))
    assert -(-most // width) * width > 2 ** 31 - 1024
    lib = library("fp4_attention")
    assert lib.gb_fp4_attention(16, hd, 16, hd, ops.BF16, 4, 16, 16, 16, 1, most, 64, 16, 4, 4, 16, 16, 8, 1, 1, hd, 16, 0.1, 0, None, 0, None) == 1
    assert b"too many rows" in lib.gb_last_error()
