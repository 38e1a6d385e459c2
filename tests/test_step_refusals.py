"""What the step's entries refuse, on the CPU: everything the slots say is checked before memory is touched, so a call
that is right in all of that ends at its host memory ("not a device pointer")."""

from __future__ import annotations

import pytest
import torch

from kernelcode_generate_amd import native

I32 = torch.int32


def assign_args(batch=3, per=4, tokens=10, stack=8):
    def ints(*shape):
        return torch.zeros(*shape, dtype=I32)

    return {"slots": torch.zeros(tokens, dtype=torch.int64), "positions": ints(tokens), "starts": ints(batch + 1),
            "page_table": ints(batch, per), "free_pages": ints(stack), "free_count": ints(1), "context_lens": ints(batch),
            "new_lens": ints(batch), "page_size": 16}


def release_args():
    a = assign_args()
    return {"page_table": a["page_table"], "free_pages": a["free_pages"], "free_count": a["free_count"], "keep_lens": a["context_lens"],
            "held_lens": a["new_lens"], "page_size": 16}


def rows_args(model=torch.bfloat16):
    return {"codes": torch.zeros(5, 16, dtype=torch.int8), "scale": torch.zeros(5), "x": torch.zeros(5, 16, dtype=model)}


def int8_args(model=torch.bfloat16, codes=True):
    return {"out": torch.zeros(5, 24, dtype=model), "x": torch.zeros(5, 16, dtype=torch.int8 if codes else model),
            "x_scale": torch.zeros(5) if codes else None, "weight": torch.zeros(24, 16, dtype=torch.int8), "w_scale": torch.zeros(24),
            "bias": None}


def rotate_args(model=torch.bfloat16):
    q, k = torch.zeros(5, 4, 64, dtype=model), torch.zeros(5, 2, 64, dtype=model)
    return {"q_out": q.clone(), "k_out": k.clone(), "q": q, "k": k, "q_weight": torch.ones(64), "k_weight": torch.ones(64, dtype=model),
            "cos": torch.ones(9, 32), "sin": torch.zeros(9, 32), "positions": torch.zeros(5, dtype=I32), "eps": 1e-6, "neighbours": False}


CALLS = {"assign": (native.kv_cache_assign, assign_args), "release": (native.kv_cache_release, release_args),
         "rows": (native.quantize_rows, rows_args), "int8": (native.int8_matmul, int8_args),
         "rotate": (native.head_norm_rotate, rotate_args)}


def refused(op, status, text, make=None, **changes):
    call, maker = CALLS[op]
    args = (make or maker)()
    assert set(changes) <= set(args)
    args.update(changes)
    with pytest.raises(native.NativeLibraryError, match=text) as caught:
        call(*args.values())
    assert caught.value.status == status


@pytest.mark.parametrize("op", sorted(CALLS))
@pytest.mark.parametrize("model", [torch.float32, torch.float16, torch.bfloat16])
def test_a_right_call_ends_at_its_host_memory(op, model):
    call, make = CALLS[op]
    makes = [make] if op in ("assign", "release") else [lambda: make(model)]
    if op == "int8":
        makes.append(lambda: make(model, codes=False))
    for one in makes:
        with pytest.raises(native.NativeLibraryError, match="not a device pointer") as caught:
            call(*one().values())
        assert caught.value.status == -1


@pytest.mark.parametrize("op", sorted(CALLS))
def test_wrong_arity_and_kind(op):
    entry = f"kg_gfx950_{CALLS[op][0].__name__}_entry"
    assert native.call_entry(entry, (1, 2), check=False) == -1
    assert "expects" in native.last_error()
    assert native.load_library()[entry](None, 0) == -1
    args = list(CALLS[op][1]().values())
    args = [int(a) if isinstance(a, bool) else a for a in args]
    for position, arg in enumerate(args):
        if isinstance(arg, torch.Tensor) or arg is None:
            wrong = [*args[:position], 3, *args[position + 1 :]]
            assert native.call_entry(entry, wrong, check=False) == -1
            assert "expected memory slot" in native.last_error()
        else:
            wrong = [*args[:position], args[0], *args[position + 1 :]]
            assert native.call_entry(entry, wrong, check=False) == -1
            assert "expected int slot" in native.last_error() or "expected float slot" in native.last_error()


@pytest.mark.parametrize("op, first, second", [("assign", "context_lens", "new_lens"), ("release", "keep_lens", "held_lens")])
def test_pages(op, first, second):
    refused(op, -1, "free_count must have one value", free_count=torch.zeros(2, dtype=I32))
    refused(op, -1, "a value for each of 3 requests", **{first: torch.zeros(2, dtype=I32)})
    refused(op, -1, "a value for each of 3 requests", **{second: torch.zeros(4, dtype=I32)})
    refused(op, -1, "unsupported dtype_code 4", **{first: torch.zeros(3, dtype=torch.int64)})
    refused(op, -1, "unsupported dtype_code 4", page_table=torch.zeros(3, 4, dtype=torch.int64))
    refused(op, -1, "expected rank 2, got 1", page_table=torch.zeros(3, dtype=I32))
    for size in (0, -1, 2**31):
        refused(op, -1, "page_size", page_size=size)
    many = torch.zeros(8193, dtype=I32)
    extra = {"starts": torch.zeros(8194, dtype=I32)} if op == "assign" else {}
    refused(op, -3, "8193 requests > 8192", page_table=torch.zeros(8193, 1, dtype=I32), **{first: many, second: many}, **extra)
    refused(op, -3, "more than 2147479552 entries", page_table=torch.zeros(3, 1, dtype=I32).expand(3, 2**30))


def test_assign():
    refused("assign", -1, "9 positions for 10 slots", positions=torch.zeros(9, dtype=I32))
    refused("assign", -1, "starts must have 4 values", starts=torch.zeros(3, dtype=I32))
    refused("assign", -1, "unsupported dtype_code 3", slots=torch.zeros(10, dtype=I32))
    long = native.TensorSpec((2**31 - 4095,), "int64", (0,)), native.TensorSpec((2**31 - 4095,), "int32", (0,))
    refused("assign", -3, "more than 2147479552 rows", slots=long[0], positions=long[1])


def test_rows():
    refused("rows", -1, "codes shape", codes=torch.zeros(5, 15, dtype=torch.int8))
    refused("rows", -1, "4 scales for 5 rows", scale=torch.zeros(4))
    refused("rows", -1, "unsupported dtype_code 6", scale=torch.zeros(5, dtype=torch.bfloat16))
    refused("rows", -1, "unsupported dtype_code 7", x=torch.zeros(5, 16, dtype=torch.int8))
    refused("rows", -1, "rows of codes and x", x=torch.zeros(5, 32)[:, ::2])


def test_int8():
    refused("int8", -1, "x K=16 != weight K=15", weight=torch.zeros(24, 15, dtype=torch.int8))
    refused("int8", -1, "out shape", out=torch.zeros(5, 23))
    refused("int8", -1, "x must be int8 or of out's type", x=torch.zeros(5, 16))
    refused("int8", -1, "needs x_scale", x_scale=None)
    refused("int8", -1, "takes no x_scale", make=lambda: int8_args(codes=False), x_scale=torch.zeros(5))
    refused("int8", -1, "4 x_scale values for 5 rows", x_scale=torch.zeros(4))
    refused("int8", -1, "23 w_scale values for 24", w_scale=torch.zeros(23))
    refused("int8", -1, "bias extent", bias=torch.zeros(23))
    refused("int8", -1, "bias dtype f16", bias=torch.zeros(24, dtype=torch.float16))
    refused("int8", -1, "unsupported dtype_code 6", weight=torch.zeros(24, 16, dtype=torch.bfloat16))
    refused("int8", -1, "rows of out, x and weight", weight=torch.zeros(24, 32, dtype=torch.int8)[:, ::2])
    refused("int8", -3, "sums may leave 32 bits", x=torch.zeros(5, 131072, dtype=torch.int8), weight=torch.zeros(24, 131072, dtype=torch.int8))


def test_rotate():
    bf16 = torch.bfloat16
    refused("rotate", -1, "q/q_out shape mismatch at dim 1", q_out=torch.zeros(5, 3, 64, dtype=bf16))
    refused("rotate", -1, "same tokens and head dim", k=torch.zeros(4, 2, 64, dtype=bf16), k_out=torch.zeros(4, 2, 64, dtype=bf16))
    refused("rotate", -1, "dtypes must match", k=torch.zeros(5, 2, 64), k_out=torch.zeros(5, 2, 64))
    refused("rotate", -1, "rows of q, k", q=torch.zeros(5, 4, 128, dtype=bf16)[..., ::2])
    refused("rotate", -1, "weight extent 63", q_weight=torch.ones(63))
    refused("rotate", -1, "weight dtype f16", k_weight=torch.ones(64, dtype=torch.float16))
    refused("rotate", -1, "cos/sin shapes", sin=torch.zeros(9, 31))
    refused("rotate", -1, "33 pairs are more", cos=torch.zeros(9, 33), sin=torch.zeros(9, 33))
    refused("rotate", -1, "4 positions for 5", positions=torch.zeros(4, dtype=I32))
    refused("rotate", -1, "unsupported dtype_code 6", cos=torch.zeros(9, 32, dtype=bf16))
    for eps in (-1e-6, float("nan"), float("inf")):
        refused("rotate", -1, "eps must be finite", eps=eps)
    args = rotate_args()
    args["neighbours"] = 2
    assert native.call_entry("kg_gfx950_head_norm_rotate_entry", list(args.values()), check=False) == -1
    assert "neighbours must be 0 or 1" in native.last_error()
    wide = torch.zeros(5, 2, 513, dtype=bf16)
    refused("rotate", -3, "head dim 513", q=wide, k=wide, q_out=wide.clone(), k_out=wide.clone(), q_weight=None, k_weight=None)


def test_no_rows_need_no_memory():
    """Tensors without elements have no memory: a call of no rows is refused for nothing that they lack."""

    args = int8_args()
    args.update(out=torch.zeros(0, 24, dtype=torch.bfloat16), x=torch.zeros(0, 16, dtype=torch.int8), x_scale=torch.zeros(0))
    with pytest.raises(native.NativeLibraryError, match="weight: data is not a device pointer"):
        native.int8_matmul(*args.values())
