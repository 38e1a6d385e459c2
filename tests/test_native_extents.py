"""What an entry sees of its tensors' extents is what they were when the call was made, whatever another thread makes of a tensor's
view meanwhile."""

from __future__ import annotations

import ctypes

import pytest
import torch

from kernelcode_generate_amd import native

native.load_library()
kg_call = pytest.importorskip("kernelcode_generate_amd._kg_call")


def seen_after(change, args):
    """[(shape, strides)] of the memory slots as the entry finds them after `change`, which runs while the entry does."""

    got = []

    def entry(slots, count):
        change()
        got.extend((s.shape[: max(s.rank, 1)], s.stride[: max(s.rank, 1)]) for s in (slots[i] for i in range(count)) if s.kind == 1)
        return 0

    kept = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.POINTER(native.KgArgSlot), ctypes.c_ulonglong)(entry)
    return got if kg_call.call(ctypes.cast(kept, ctypes.c_void_p).value, args) == 0 else None


def test_extents_are_the_calls_own():
    x, y, scalar = torch.zeros(4, 6), torch.zeros(3, 5, 7), torch.tensor(1.0)
    want = [([4, 6], [6, 1]), ([3, 5, 7], [35, 7, 1]), ([0], [0]), ([0], [1])]
    assert seen_after(lambda: None, (x, y, 3, scalar, None)) == want
    assert seen_after(lambda: (x.t_(), y.transpose_(0, 2)), (x, y, 3, scalar, None)) == want
    assert x.shape == (6, 4) and y.shape == (7, 5, 3)


def test_more_axes_than_any_entry_takes_are_left_to_python():
    assert seen_after(lambda: None, (torch.zeros([1] * 8),)) == [([1] * 8, [1] * 8)]
    assert seen_after(lambda: None, (torch.zeros([1] * 9),)) is None
    with pytest.raises(native.NativeLibraryError, match="expected rank 2, got 9"):
        native.quantize_rows(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4), torch.zeros([1] * 9))
