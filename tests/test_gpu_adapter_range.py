"""x A of an adapter times its scale may leave fp16's range at either end while the output stays inside it: against 64 bits,
in every form of the projection and in the general one (operands that are not aligned)."""

from __future__ import annotations

import pytest
import torch

from tests.serving_util import adapter_oracle, assert_rows
from tests.test_gpu_adapter_matmul import Call
from kernelcode_generate_amd import native

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
# m, k, n, adapters, rank: few rows, 128 x 128 tiles, a split K, ragged and whole wide tiles, rank in more than one block of 64 columns
SHAPES = [(1, 512, 512, 2, 16), (33, 2048, 320, 3, 64), (400, 256, 384, 4, 136), (520, 512, 640, 5, 16), (600, 2048, 256, 3, 8),
          (4104, 544, 2056, 3, 16), (4096, 544, 2048, 3, 16)]


def shifted(t):
    return torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].reshape(t.shape)


@pytest.mark.parametrize("model", [F16, BF16])
@pytest.mark.parametrize("aligned,m,k,n,count,rank", [(True, *s) for s in SHAPES] + [(False, *s) for s in SHAPES[:5]])
def test_large_and_small_sums(device, aligned, m, k, n, count, rank, model):
    """Adapter l's t of some 2^17 (B of some 2^-17 beside it), 1, or 2^-20 (B of some 2^13), by l % 3."""

    call = Call(m, k, n, count, rank, model, bias=torch.float32, order="sorted")
    call.index = torch.arange(m, dtype=torch.int32) % count
    call.scale = torch.ones(count)
    call.w = (call.w.float() * 0.25).to(model)
    b = call.b.float()
    for l in range(count):
        power = (17, 0, -20)[l % 3]
        call.scale[l] = 1.3 * 2.0**power
        b[l] *= 2.0 ** min(-power, 13)
    call.b = b.to(model)  # (what has no fp16 value is the nearest one: an operand like any other)
    args = call.args(device)
    if not aligned:
        args[0] = shifted(args[0])
    out = torch.full((m, n), 9.0, dtype=model, device=device)
    native.adapter_matmul(out, *args)
    assert torch.isfinite(out).all()
    call.check(out)


@pytest.mark.parametrize("m,k,n,count,rank", SHAPES)
def test_the_projection_beside_extreme_sums(device, m, k, n, count, rank):
    """B of zeros: the projection's own result, whatever t is (2^100, 2^-100, 0), within half a step of the type."""

    call = Call(m, k, n, 3, rank, F16, bias=torch.float32)
    call.index = torch.arange(m, dtype=torch.int32) % 3
    call.scale = torch.tensor([2.0**100, 2.0**-100, 0.0])
    call.b[:] = 0.0
    call.check(call.run(device))


def test_rows_that_are_infinite(device):
    """A sum past 32 bits is infinite, and so is the row; finite sums beside it change nothing about that."""

    call = Call(6, 64, 64, 2, 16, F16)
    call.index = torch.tensor([0, 1, 0, 1, -1, 1], dtype=torch.int32)
    call.scale = torch.tensor([1.0, 3e38])
    call.x = call.x.abs()
    call.a[1] = 1000.0
    call.a[1, :, 3] = 1e-4
    call.b[:] = call.b.abs()
    out = call.run(device)
    rows = call.index == 1
    assert torch.isposinf(out[rows.to(device)]).all()
    keep = torch.nonzero(~rows).flatten()
    expected, allowed = adapter_oracle(call.x[keep], call.w, None, call.a, call.b, call.index[keep], torch.tensor([1.0, 1.0]))
    assert_rows(out[keep.to(device)], expected, allowed)
