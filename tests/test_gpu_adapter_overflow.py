"""fp16 rows whose projection alone is past the type's range while the sum with the adapter is not: the formula's finite value, whatever
the operands' alignment."""

from __future__ import annotations

import pytest
import torch

from kernelcode_generate_amd import native
from tests.serving_util import adapter_oracle, assert_rows
from tests.test_gpu_adapter_matmul import Call

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def shifted(t):
    return torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].reshape(t.shape)


@pytest.mark.parametrize("bias", [None, F32, F16])
@pytest.mark.parametrize("m,k,n,count,rank,layout", [
    (5, 128, 96, 2, 8, "aligned"), (5, 128, 96, 2, 8, "shifted"), (700, 256, 264, 2, 16, "aligned"), (300, 256, 264, 2, 16, "shifted"),
    (9, 37, 41, 2, 5, "aligned"), (70, 129, 65, 2, 1, "aligned"), (6, 130, 64, 2, 3, "columns"),  # weight and bias of every second column
])
def test_projections_past_the_range(device, m, k, n, count, rank, layout, bias):
    call = Call(m, k, n, count, rank, F16, bias=bias, scaled=False)
    call.index = torch.arange(m, dtype=torch.int32) % 3 - 1
    call.x = (call.x.abs() + 0.5).half()
    call.x[0] = 0.25
    call.w = torch.full((k, n), 90000.0 / k).half()  # sums of some 90000 and more
    call.w[:, ::2] *= -1
    call.a = torch.full((count, k, rank), 1.0 / k).half()
    call.b = torch.full((count, rank, n), -60000.0 / rank).half()  # brings them back
    call.b[:, :, ::2] *= -1
    x, w, b, a, low, index, scale = call.args(device)
    if layout == "shifted":
        x = shifted(x)
    elif layout == "columns":
        w = torch.stack([w, torch.zeros_like(w)], -1).reshape(k, 2 * n)[:, ::2]
        b = None if b is None else torch.stack([b, torch.zeros_like(b)], -1).reshape(-1)[::2]
    out = torch.full((m, n), 9.0, dtype=F16, device=device)
    native.adapter_matmul(out, x, w, b, a, low, index, scale)
    expected, allowed = adapter_oracle(call.x, call.w, call.bias, call.a, call.b, call.index, call.scale)
    # past the range by more than the error allowed: an infinity; within it by more: the value; between: either
    top = 65520.0  # rounds to an infinity
    inside, outside = abs(expected) + allowed < top, abs(expected) - allowed >= top
    got = out.cpu()
    rows = (call.index >= 0)[:, None].numpy()
    assert (inside & rows).any()
    import numpy as np

    assert_rows(torch.where(torch.from_numpy(inside), got, torch.zeros_like(got)), np.where(inside, expected, 0.0), np.where(inside, allowed, 0.0))
    assert torch.isinf(got[torch.from_numpy(outside)]).all()
