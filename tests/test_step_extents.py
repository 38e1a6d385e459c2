"""Calls whose extents no memory has: axes without strides, rows on one another, whose work would not end. They are refused before memory is
touched; a call as large as a card's memory can hold is not."""

from __future__ import annotations

import pytest

from kernelcode_generate_amd import native
from kernelcode_generate_amd.native import TensorSpec

MOST = 2**31 - 1


def spec(dtype, *shape, strides=None):
    return TensorSpec(shape, dtype, strides if strides is not None else (0,) * (len(shape) - 1) + (1,))


def outcome(entry, *args):
    status = native.call_entry(f"kg_gfx950_{entry}_entry", args, check=False)
    return status, native.last_error()


@pytest.mark.parametrize("m, k, refused", [(MOST, 4096, True), (2**27 + 1, 4096, True), (2**27, 4096, False), (MOST, 64, False), (256, 2147418112, False)])
def test_quantize_rows(m, k, refused):
    status, text = outcome("quantize_rows", spec("int8", m, k), spec("float32", m, strides=(0,)), spec("bfloat16", m, k))
    assert (status, "elements" in text) == ((-3, True) if refused else (-1, False)), text
    assert refused or "not a device pointer" in text


@pytest.mark.parametrize("m, n, k, refused", [(MOST, MOST, 1, True), (MOST, 256, 8, True), (MOST, 128, 8, False), (2**19, 2**19 + 1, 131071, True), (2**19, 2**19, 131071, False)])
@pytest.mark.parametrize("x", ["int8", "float16"])
def test_int8_matmul(m, n, k, refused, x):
    args = (spec("float16", m, n), spec(x, m, k), spec("float32", m, strides=(0,)) if x == "int8" else None, spec("int8", n, k),
            spec("float32", n, strides=(0,)), None)
    status, text = outcome("int8_matmul", *args)
    assert (status, "results" in text) == ((-3, True) if refused else (-1, False)), text
    assert refused or "not a device pointer" in text
    if refused:
        with pytest.raises(native.NativeLibraryError, match="results"):
            native.cost("int8_matmul", args)


@pytest.mark.parametrize("t, heads, d, refused", [(MOST, MOST, 512, True), (MOST, MOST, 1, True), (2**20, 2**9 + 1, 512, True), (2**20, 2**9, 512, False),
                                                  (MOST, 128, 1, False)])
def test_head_norm_rotate(t, heads, d, refused):
    rows, none = spec("bfloat16", t, heads, d), spec("bfloat16", t, 0, d)
    table = TensorSpec((4, 0), "float32")
    status, text = outcome("head_norm_rotate", rows, none, rows, none, None, None, table, table, spec("int32", t, strides=(0,)), 1e-6, 0)
    assert (status, "elements" in text) == ((-3, True) if refused else (-1, False)), text
    assert refused or "not a device pointer" in text
