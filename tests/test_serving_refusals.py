"""What the serving entries refuse, on the CPU: everything the slots say is checked before memory is touched, so
a call that is right in all of that ends at its host memory ("not a device pointer")."""

from __future__ import annotations

import pytest
import torch

from kernelcode_generate_amd import native

E4M3 = torch.float8_e4m3fn


def store_args(cache=torch.bfloat16, model=torch.bfloat16, pages=3, heads=2, page=16, d=64, tokens=5):
    caches = [torch.zeros(pages, heads, page, d).to(cache) for _ in range(2)]
    scales = [torch.zeros(pages, heads, page) if cache in (torch.int8, E4M3) else None for _ in range(2)]
    rows = [torch.zeros(tokens, heads, d, dtype=model) for _ in range(2)]
    return dict(zip(("k_cache", "v_cache", "k_scale", "v_scale", "k", "v", "slots"),
                    [*caches, *scales, *rows, torch.zeros(tokens, dtype=torch.int64)]))


def load_args(cache=torch.bfloat16, model=torch.bfloat16, batch=2, rows=9):
    a = store_args(cache, model)
    outs = [torch.zeros(batch, 2, rows, 64, dtype=model) for _ in range(2)]
    return {"k_out": outs[0], "v_out": outs[1], **{x: a[x] for x in ("k_cache", "v_cache", "k_scale", "v_scale")},
            "page_table": torch.zeros(batch, 1, dtype=torch.int32), "lengths": torch.zeros(batch, dtype=torch.int32)}


def tree_args(cache=torch.bfloat16, model=torch.bfloat16, batch=2, tokens=5, heads_q=4, mask=False):
    a = load_args(cache, model, batch)
    q = torch.zeros(tokens, heads_q, 64, dtype=model)
    return {"out": q.clone(), "q": q, **{x: a[x] for x in ("k_cache", "v_cache", "k_scale", "v_scale", "page_table")},
            "context_lens": torch.zeros(batch, dtype=torch.int32), "starts": torch.zeros(batch + 1, dtype=torch.int32),
            "mask": torch.zeros(tokens, 1, dtype=torch.int64) if mask else None, "scale": 1.0}


def adapter_args(model=torch.bfloat16, m=5, k=16, n=24, adapters=3, rank=8):
    return {"out": torch.zeros(m, n, dtype=model), "x": torch.zeros(m, k, dtype=model), "weight": torch.zeros(k, n, dtype=model),
            "bias": None, "a": torch.zeros(adapters, k, rank, dtype=model), "b": torch.zeros(adapters, rank, n, dtype=model),
            "index": torch.zeros(m, dtype=torch.int32), "scale": torch.ones(adapters)}


CALLS = {"store": (native.kv_cache_store, store_args), "load": (native.kv_cache_load, load_args),
         "tree": (native.tree_attention, tree_args), "adapter": (native.adapter_matmul, adapter_args)}


def refused(op, make, status, text, **changes):
    call, _ = CALLS[op]
    args = make()
    assert set(changes) <= set(args)
    args.update(changes)
    with pytest.raises(native.NativeLibraryError, match=text) as caught:
        call(*args.values())
    assert caught.value.status == status


@pytest.mark.parametrize("op", sorted(CALLS))
@pytest.mark.parametrize("model", [torch.float32, torch.float16, torch.bfloat16])
def test_a_right_call_ends_at_its_host_memory(op, model):
    call, make = CALLS[op]
    caches = (None,) if op == "adapter" else (model, torch.int8, E4M3)
    for cache in caches:
        args = make(model=model) if cache is None else make(cache, model)
        with pytest.raises(native.NativeLibraryError, match="not a device pointer") as caught:
            call(*args.values())
        assert caught.value.status == -1


@pytest.mark.parametrize("op", sorted(CALLS))
def test_wrong_arity_and_kind(op):
    entry = CALLS[op][0].__name__
    assert native.call_entry(f"kg_gfx950_{entry}_entry", (1, 2), check=False) == -1
    assert "expects" in native.last_error()
    assert native.load_library()[f"kg_gfx950_{entry}_entry"](None, 0) == -1
    args = list(CALLS[op][1]().values())
    for position in range(len(args) - (op == "tree")):
        wrong = [*args[:position], 3, *args[position + 1 :]]
        assert native.call_entry(f"kg_gfx950_{entry}_entry", wrong, check=False) == -1
        assert "expected memory slot" in native.last_error()


def test_caches():
    bf16, f16 = torch.bfloat16, torch.float16
    for op in ("store", "load", "tree"):
        make = CALLS[op][1]
        refused(op, make, -1, "dtypes must match", v_cache=torch.zeros(3, 2, 16, 64, dtype=f16))
        refused(op, make, -1, "shape mismatch at dim 0", v_cache=torch.zeros(2, 2, 16, 64, dtype=bf16))
        refused(op, make, -1, "takes no scales", k_scale=torch.zeros(3, 2, 16))
        refused(op, make, -1, "rows of a cache must be contiguous", k_cache=torch.zeros(3, 2, 16, 128, dtype=bf16)[..., ::2])
        refused(op, make, -1, "expected rank 4, got 3", k_cache=torch.zeros(3, 2, 16, dtype=bf16))
        refused(op, make, -1, "unsupported dtype_code 3", k_cache=torch.zeros(3, 2, 16, 64, dtype=torch.int32))
        refused(op, make, -1, "expected memory slot|memory slot has no data|expected rank", k_cache=None)
        for cache in (torch.int8, E4M3):
            make8 = lambda: CALLS[op][1](cache)  # noqa: E731
            refused(op, make8, -1, "needs k_scale and v_scale", v_scale=None)
            refused(op, make8, -1, "cache/scale shape mismatch at dim 2", k_scale=torch.zeros(3, 2, 15))
            refused(op, make8, -1, "unsupported dtype_code 6", k_scale=torch.zeros(3, 2, 16, dtype=bf16))
    refused("store", store_args, -3, "head dim 513", k_cache=torch.zeros(3, 2, 16, 513, dtype=bf16),
            v_cache=torch.zeros(3, 2, 16, 513, dtype=bf16))
    refused("store", store_args, -1, "at least one token", k_cache=torch.zeros(3, 2, 0, 64, dtype=bf16),
            v_cache=torch.zeros(3, 2, 0, 64, dtype=bf16))


def test_store():
    rows = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    refused("store", store_args, -1, "must be .tokens, 2, 64.", k=rows[:, :1])
    refused("store", store_args, -1, "must be .tokens, 2, 64.", v=rows[:4])
    refused("store", store_args, -1, "dtypes must match", v=rows.half())
    refused("store", store_args, -1, "dtypes must match", k=rows.half(), v=rows.half())
    refused("store", store_args, -1, "rows of k and v", k=torch.zeros(5, 2, 128, dtype=torch.bfloat16)[..., ::2])
    refused("store", store_args, -1, "4 slots for 5 tokens", slots=torch.zeros(4, dtype=torch.int64))
    refused("store", store_args, -1, "unsupported dtype_code 3", slots=torch.zeros(5, dtype=torch.int32))


def test_load():
    refused("load", load_args, -1, "must be .batch, 2, rows, 64.", v_out=torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16))
    refused("load", load_args, -1, "dtypes must match", v_out=torch.zeros(2, 2, 9, 64))
    refused("load", load_args, -1, "a row for each of 2", lengths=torch.zeros(3, dtype=torch.int32))
    refused("load", load_args, -1, "a row for each of 2", page_table=torch.zeros(1, 1, dtype=torch.int32))
    refused("load", load_args, -1, "unsupported dtype_code 4", page_table=torch.zeros(2, 1, dtype=torch.int64))


def test_tree():
    bf16 = torch.bfloat16
    refused("tree", tree_args, -1, "q/out shape mismatch at dim 0", out=torch.zeros(4, 4, 64, dtype=bf16))
    refused("tree", tree_args, -1, "no multiple of 2 key heads", out=torch.zeros(5, 3, 64, dtype=bf16),
            q=torch.zeros(5, 3, 64, dtype=bf16))
    refused("tree", tree_args, -1, "head dim 32 of q", out=torch.zeros(5, 4, 32, dtype=bf16), q=torch.zeros(5, 4, 32, dtype=bf16))
    refused("tree", tree_args, -1, "dtypes must match", q=torch.zeros(5, 4, 64))
    refused("tree", tree_args, -1, "rows of q and out", q=torch.zeros(5, 4, 128, dtype=bf16)[..., ::2])
    refused("tree", tree_args, -1, "page_table has 3 rows for 2", page_table=torch.zeros(3, 1, dtype=torch.int32))
    refused("tree", tree_args, -1, "starts must have 3 values", starts=torch.zeros(2, dtype=torch.int32))
    refused("tree", tree_args, -1, "mask has 4 rows for 5", mask=torch.zeros(4, 1, dtype=torch.int64))
    refused("tree", tree_args, -1, "unsupported dtype_code 3", mask=torch.zeros(5, 1, dtype=torch.int32))
    refused("tree", tree_args, -1, "scale must be finite", scale=float("nan"))
    refused("tree", tree_args, -1, "scale must be finite", scale=1e300)
    wide = torch.zeros(2, 1, dtype=torch.int32).expand(2, 1 << 28)
    refused("tree", tree_args, -3, "exceeds int32", page_table=wide)


def test_adapter():
    bf16 = torch.bfloat16
    refused("adapter", adapter_args, -1, "x K=16 != weight K=15", weight=torch.zeros(15, 24, dtype=bf16))
    refused("adapter", adapter_args, -1, "out shape", out=torch.zeros(5, 23, dtype=bf16))
    refused("adapter", adapter_args, -1, "bias extent", bias=torch.zeros(23))
    refused("adapter", adapter_args, -1, "bias dtype f16", bias=torch.zeros(24, dtype=torch.float16))
    refused("adapter", adapter_args, -1, "a must be", a=torch.zeros(3, 15, 8, dtype=bf16))
    refused("adapter", adapter_args, -1, "b must be", b=torch.zeros(3, 7, 24, dtype=bf16))
    refused("adapter", adapter_args, -1, "b must be", b=torch.zeros(2, 8, 24, dtype=bf16))
    refused("adapter", adapter_args, -1, "4 indexes for 5 rows", index=torch.zeros(4, dtype=torch.int32))
    refused("adapter", adapter_args, -1, "2 scales for 3 adapters", scale=torch.ones(2))
    refused("adapter", adapter_args, -1, "dtypes must match", a=torch.zeros(3, 16, 8))
    refused("adapter", adapter_args, -1, "unsupported dtype_code 4", index=torch.zeros(5, dtype=torch.int64))
    refused("adapter", adapter_args, -1, "rows of out, x, a and b", x=torch.zeros(5, 32, dtype=bf16)[:, ::2])
    refused("adapter", adapter_args, -3, "rank 513 > 512", a=torch.zeros(3, 16, 513, dtype=bf16), b=torch.zeros(3, 513, 24, dtype=bf16))


def test_other_entries_take_no_8_bit_memory():
    x = torch.zeros(4, 4, dtype=torch.int8)
    with pytest.raises(native.NativeLibraryError, match="unsupported dtype_code 7"):
        native.matmul(x, x, x)


def test_axes_without_strides_are_elements():
    """Extents whose product is a multiple of 2^64 are no empty tensor: the memory behind them is checked."""

    cache = native.TensorSpec((2**30, 2**4, 2**26, 64), "bfloat16", (0, 0, 0, 1))
    refused("load", load_args, -1, "k_out: data is not a device pointer",
            **{x: native.TensorSpec((2**30, 2**4, 2**26, 64), "bfloat16", (0, 0, 0, 1)) for x in ("k_out", "v_out")},
            k_cache=cache, v_cache=cache, page_table=native.TensorSpec((2**30, 1), "int32", (0, 0)),
            lengths=native.TensorSpec((2**30,), "int32", (0,)))
    rows = native.TensorSpec((2**30, 2**30, 64), "bfloat16", (0, 0, 1))
    refused("tree", tree_args, -1, "out: data is not a device pointer", out=rows, q=rows)


def test_the_most_positions_of_a_request():
    """Past 2^31 - 4096 the kernels' steps and the pages looked up ahead would leave 32 bits."""

    for columns, page, text in ((2**27 - 256, 16, "not a device pointer"), (2**27 - 255, 16, "exceeds int32")):
        caches = [torch.zeros(1, 2, page, 64, dtype=torch.bfloat16) for _ in range(2)]
        refused("tree", tree_args, -1 if text.startswith("not") else -3, text, k_cache=caches[0], v_cache=caches[1],
                page_table=torch.zeros(2, 1, dtype=torch.int32).expand(2, columns))
