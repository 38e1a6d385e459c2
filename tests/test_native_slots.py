"""How call arguments become slots: what an object is counts, not what another object of its class was."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from kernelcode_generate_amd import native


def memory_like():
    return SimpleNamespace(data_ptr=lambda: 64, shape=(2, 3), stride=lambda: (3, 1), dtype="float32")


def test_objects_of_one_class():
    """One with a memory argument's attributes of its own does not make another one memory."""

    slots, _ = native.marshal_slots([memory_like()])
    assert (slots[0].kind, slots[0].rank, slots[0].dtype_code, slots[0].shape[1], slots[0].stride[0]) == (1, 2, 1, 3, 3)
    with pytest.raises(native.NativeLibraryError, match="unsupported runtime arg at position 1: SimpleNamespace"):
        native.marshal_slots([memory_like(), SimpleNamespace(shape=(2,))])


def test_subclasses_and_specs():
    class Own(torch.Tensor):
        pass

    for x in (torch.zeros(4, 5).as_subclass(Own), torch.nn.Parameter(torch.zeros(4, 5)), native.TensorSpec((4, 5), "float32")):
        slots, _ = native.marshal_slots([x, 7, 1.5])
        assert (slots[0].rank, slots[0].shape[0], slots[0].shape[1], slots[0].stride[0], slots[0].stride[1]) == (2, 4, 5, 5, 1)
        assert slots[0].data == x.data_ptr() and slots[1].int_value == 7 and slots[2].float_value == 1.5
