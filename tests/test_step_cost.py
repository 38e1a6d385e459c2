"""native.cost of int8_matmul, without a GPU."""

from __future__ import annotations

import pytest

from kernelcode_generate_amd import native
from kernelcode_generate_amd.native import TensorSpec as T


def cost(m, n, k, x="int8", out="bfloat16", bias=None, pitch=None):
    pitch = pitch or k
    args = (T((m, n), out), T((m, k), x, (pitch, 1)), T((m,), "float32") if x == "int8" else None, T((n, k), "int8", (pitch, 1)),
            T((n,), "float32"), None if bias is None else T((n,), bias))
    return native.cost("int8_matmul", args)


def test_codes():
    c = cost(4096, 4096, 4096)
    assert c["MAC"] == 4096**3
    assert c["MFMA"] * 16 * 16 * 64 == 4096**3  # whole tiles: nothing but the product's own
    assert c["MFMA_CYCLES"] == 16 * c["MFMA"]
    assert c["HBM_READ"] == 2 * 4096**2 + 2 * 4 * 4096 and c["HBM_WRITE"] == 2 * 4096**2
    c = cost(1000, 1501, 1024, out="float32", bias="float32")
    assert c["MAC"] == 1000 * 1501 * 1024 and c["MFMA"] * 16 * 16 * 64 >= c["MAC"]
    assert c["HBM_READ"] == (1000 + 1501) * 1024 + 4 * 1501 * 2 + 4 * 1000 and c["HBM_WRITE"] == 4 * 1000 * 1501


def test_rows_that_the_call_quantises():
    c = cost(300, 4096, 4096, x="bfloat16")
    assert c["HBM_READ"] == 300 * 4096 * 2 + 4096**2 + 4 * 4096 + 300 * 4096  # the codes are written and read
    assert c["HBM_WRITE"] == 300 * 4096 * 2 + 300 * 4096


def test_weights_of_no_whole_pieces():
    assert cost(300, 512, 1023)["HBM_WRITE"] == 300 * 512 * 2 + (300 + 512) * 1024
    assert cost(16, 512, 8)["MFMA"] == 0  # the general kernel


def test_few_tiles_of_a_long_k():
    """The sums of the chunks of K, four bytes each, are written and read; the products are those of one chunk."""

    c = cost(16, 500, 16384)
    base = 16 * 500 * 2
    chunks = (c["HBM_WRITE"] - base) / (16 * 500 * 4)
    assert chunks in (2, 4, 8)
    assert c["HBM_READ"] == (16 + 500) * 16384 + 4 * 500 + 4 * 16 + c["HBM_WRITE"] - base
    assert c["MFMA"] % (16384 // 64) == 0 and c["MFMA"] * 16 * 16 * 64 >= c["MAC"]
    assert cost(4096, 4096, 16384)["HBM_WRITE"] == 2 * 4096**2  # many tiles: none


def test_refusals_are_the_entry_s():
    with pytest.raises(native.NativeLibraryError, match="sums may leave 32 bits"):
        cost(4, 4, 131072)
    assert cost(0, 8, 64)["MAC"] == 0
