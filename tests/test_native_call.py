"""The host module that calls an entry with torch tensors: the slots that it packs are marshal_slots', and what it does not know it
leaves to Python."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from kernelcode_generate_amd import native

native.load_library()
kg_call = pytest.importorskip("kernelcode_generate_amd._kg_call")


def words(slots, count):
    def axis(pointer, rank):
        return [pointer[i] for i in range(max(rank, 1))]

    return [(s.kind, s.data, axis(s.shape, s.rank) if s.shape else None, axis(s.stride, s.rank) if s.stride else None, s.rank, s.dtype_code,
             s.int_value, s.float_value) for s in (slots[i] for i in range(count))]


def seen_by_an_entry(args):
    """(status, the slots that an entry gets)."""

    got = []
    entry = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.POINTER(native.KgArgSlot), ctypes.c_ulonglong)(
        lambda slots, count: got.append(words(slots, count)) or 7)
    status = kg_call.call(ctypes.cast(entry, ctypes.c_void_p).value, args)
    return status, got[0] if got else None


def test_slots_are_marshal_slots_own():
    x = torch.arange(120, dtype=torch.float32).reshape(4, 5, 6)
    args = (x, x[1:, ::2, 3:], x.transpose(0, 2), None, 3, -(2**63), 2**63 - 1, 0.5, float("-inf"), torch.tensor(2.0, dtype=torch.bfloat16),
            torch.zeros(0, 7), torch.zeros(3, 0, dtype=torch.int32), x.half()[0].expand(9, 5, 6), torch.nn.Parameter(torch.ones(3)),
            torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int8), torch.zeros(2).to(torch.float8_e4m3fn), torch.zeros(2, dtype=torch.float64))
    status, got = seen_by_an_entry(args)
    assert status == 7
    slots, keep = native.marshal_slots(args)
    want = words(slots, len(args))
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert a == b
    del keep


def test_a_lazy_copy_is_made_before_an_entry_writes_it():
    x = torch.ones(40)
    y = torch._lazy_clone(x)  # shares x's memory until either is written
    _, got = seen_by_an_entry((y,))
    assert got[0][1] == y.data_ptr() != x.data_ptr()


class Odd(torch.Tensor):
    pass


@pytest.mark.parametrize("odd", [True, np.int32(3), np.float32(0.5), 2**63, "x", np.zeros(3, np.float32), native.TensorSpec((3,), "float32"),
                                 torch.zeros(3, dtype=torch.int16), torch.zeros(3).as_subclass(Odd), torch.zeros(3, 3).to_sparse()],
                         ids=lambda v: type(v).__name__)
def test_what_is_not_known_is_left_to_python(odd):
    assert seen_by_an_entry((torch.zeros(3), odd)) == (None, None)


def test_no_more_slots_than_it_has():
    assert seen_by_an_entry((1,) * 32)[0] == 7
    assert seen_by_an_entry((1,) * 33) == (None, None)
    assert seen_by_an_entry(()) == (7, [])
    with pytest.raises(TypeError):
        kg_call.call(1)
    with pytest.raises(TypeError):
        kg_call.call("x", ())


def test_call_entry_reports_the_same_either_way(monkeypatch):
    x = torch.zeros(4, 16)
    texts = []
    for fast in (native._FAST_CALL, None):
        monkeypatch.setattr(native, "_FAST_CALL", fast)
        for args in ((x.to(torch.int8), torch.zeros(4), x), (x, torch.zeros(4), x), (x, x), (3, x, x), (x.to(torch.int8), True, x),
                     (x.to(torch.int8), np.int64(4), x), (x.to(torch.int16), torch.zeros(4), x)):
            with pytest.raises(native.NativeLibraryError) as caught:
                native.call_entry("kg_gfx950_quantize_rows_entry", args)
            texts.append((str(caught.value), caught.value.status))
    assert texts[:7] == texts[7:]
