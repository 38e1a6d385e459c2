"""Which tiles and chunks of K int8_matmul takes for a call, read from native.cost: it counts the matrix instructions of the tiles and the
bytes of a split K's sums."""

from __future__ import annotations

import itertools

from kernelcode_generate_amd import native
from kernelcode_generate_amd.native import TensorSpec

# (rows, channels, stages of the ring) of the tiles
FORMS = ((256, 256, 2), (256, 128, 3), (128, 128, 4), (128, 64, 3), (64, 64, 4), (32, 64, 4), (32, 32, 8))
SPLIT_FORMS = FORMS[4:]
WORKSPACE = 64 << 20
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


def up(x: int, unit: int) -> int:
    return -(-x // unit) * unit


def instructions(form, m: int, n: int, k: int, chunk: int) -> int:
    """16 x 16 x 64 products of one piece: whole tiles, whole slices of 128 k, at least a ring of them."""

    rows, channels, stages = form
    slices = sum(max(up(min(chunk, k - at), 128) // 128, stages) for at in range(0, k, chunk))
    return (up(m, rows) // 16) * (up(n, channels) // 16) * 2 * slices


def chosen(m: int, n: int, k: int, codes: bool, out: str = "bfloat16") -> tuple[list, int]:
    """(the forms that its pieces may have taken, a tuple for each reading of the cost; chunks of K). One piece of channels."""

    whole, pitch = k % 16 == 0, up(k, 64)
    args = (TensorSpec((m, n), out), TensorSpec((m, k), "int8" if codes else out), TensorSpec((m,), "float32") if codes else None,
            TensorSpec((n, k), "int8"), TensorSpec((n,), "float32"), None)
    cost = native.cost("int8_matmul", args)
    w_bytes, row_bytes = 0 if whole else n * pitch, 0 if codes and whole else pitch + (0 if codes else 4)
    assert w_bytes <= WORKSPACE // 2
    rows = m if row_bytes == 0 else min(m, max(128, (WORKSPACE - w_bytes - 1024) // row_bytes // 128 * 128))
    sums = cost["HBM_WRITE"] - m * n * BYTES[out] - w_bytes - (m * pitch if row_bytes else 0)
    chunks, left = divmod(sums, m * up(n, 4) * 4)
    assert left == 0 and chunks != 1
    deep = k if whole else pitch
    if chunks:
        assert rows == m
        splits = {up(deep // s, 128) for s in (2, 4, 8)}
        found = [(form,) for form in SPLIT_FORMS for chunk in splits
                 if -(-deep // chunk) == chunks and instructions(form, m, n, deep, chunk) == cost["MFMA"]]
        return found, chunks
    parts = [min(rows, m - at) for at in range(0, m, rows)]
    kinds = sorted(set(parts), reverse=True)  # (pieces of one size take one form)
    found = []
    for forms in itertools.product(FORMS, repeat=len(kinds)):
        total = sum(instructions(forms[kinds.index(p)], p, n, deep, deep) for p in parts)
        if total == cost["MFMA"]:
            found.append(forms)
    return found, 1
