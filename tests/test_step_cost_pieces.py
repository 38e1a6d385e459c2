"""native.cost of int8_matmul calls whose copies are more than the workspace holds: what is written and read again, for each piece."""

from __future__ import annotations

import pytest

from kernelcode_generate_amd import native
from kernelcode_generate_amd.native import TensorSpec as T


def cost(m, n, k, x="int8"):
    args = (T((m, n), "bfloat16"), T((m, k), x), T((m,), "float32") if x == "int8" else None, T((n, k), "int8"), T((n,), "float32"), None)
    return native.cost("int8_matmul", args)


def pieces(n, k):
    """Pieces of channels: as many multiples of 128 as half of the 64 MiB hold, at a pitch of whole 64 bytes."""

    pitch = -(-k // 64) * 64
    return -(-n // max(128, ((32 << 20) - 1024) // pitch // 128 * 128)), pitch


@pytest.mark.parametrize("x, size", [("bfloat16", 2), ("int8", 1)])
@pytest.mark.parametrize("m, n, k, want", [(600, 5000, 16383, 3), (70, 9000, 8191, 3), (16, 512, 4095, 1), (40, 300, 131071, 3)])
def test_rows_are_made_ready_for_every_piece_of_channels(m, n, k, want, x, size):
    """Each piece of channels reads the rows and writes their codes (quantised, or copied) once more; weights are copied once."""

    count, pitch = pieces(n, k)
    assert count == want
    c = cost(m, n, k, x)
    copies = (count * m + n) * pitch
    base = m * n * 2
    sums = c["HBM_WRITE"] - base - copies
    assert sums >= 0 and sums % (m * (-(-n // 4) * 4) * 4) == 0  # of a split K: none of several pieces
    assert sums == 0 or count == 1
    assert c["HBM_READ"] == count * m * k * size + n * k + 4 * n + (4 * m if x == "int8" else 0) + copies + sums


def test_rows_in_pieces_are_made_ready_once():
    c = cost(20000, 40, 4000, "bfloat16")  # pieces of rows, one of channels
    assert c["HBM_WRITE"] == 20000 * 40 * 2 + 20000 * 4032
    assert c["HBM_READ"] == 20000 * 4000 * 2 + 40 * 4000 + 4 * 40 + 20000 * 4032
