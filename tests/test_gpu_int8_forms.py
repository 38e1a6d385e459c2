"""int8_matmul in each of its forms by name: every shape of tiles that splits K, in two, four and eight chunks, and the largest sums in every
shape of tiles with K whole. The sizes are those that the entry's model gives these forms, which is checked without a GPU: a model that
is fitted anew has to come with sizes that reach them."""

from __future__ import annotations

import pytest
import torch

from kernelcode_generate_amd import native
from tests.int8_forms import FORMS, SPLIT_FORMS, chosen
from tests.serving_util import HALF
from tests.step_util import STEP
from tests.test_gpu_int8_matmul import check_product

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# (m, n, k): (tiles, chunks); odd sizes, K of whole 16-byte pieces and not
SPLITS = {
    (65, 1037, 8368): (SPLIT_FORMS[2], 2), (118, 654, 7932): (SPLIT_FORMS[2], 2), (1, 71, 4864): (SPLIT_FORMS[2], 4), (1, 87, 4886): (SPLIT_FORMS[2], 4),
    (1, 34, 8720): (SPLIT_FORMS[2], 8), (1, 35, 7768): (SPLIT_FORMS[2], 8),
    (134, 1346, 26624): (SPLIT_FORMS[1], 2), (201, 1033, 24232): (SPLIT_FORMS[1], 2), (66, 1153, 9648): (SPLIT_FORMS[1], 4),
    (65, 1050, 10829): (SPLIT_FORMS[1], 4), (1, 1054, 13984): (SPLIT_FORMS[1], 8), (1, 1032, 14735): (SPLIT_FORMS[1], 8),
    (202, 1191, 9888): (SPLIT_FORMS[0], 2), (328, 746, 10119): (SPLIT_FORMS[0], 2), (75, 1355, 11728): (SPLIT_FORMS[0], 4),
    (65, 1361, 11612): (SPLIT_FORMS[0], 4), (66, 692, 8000): (SPLIT_FORMS[0], 8), (72, 686, 7548): (SPLIT_FORMS[0], 8),
}
LONG = 131056  # 2^14 times that is the largest sum of whole 16-byte pieces
# (m, n, rows in codes): the form of the last piece of rows (of those that the call quantises: 384 and 270 of 654)
LARGEST = {(654, 600, False): FORMS[6], (654, 1300, False): FORMS[5], (654, 2000, False): FORMS[4], (654, 5000, False): FORMS[3],
           (1630, 1300, True): FORMS[2], (1800, 3700, True): FORMS[1], (1930, 4420, True): FORMS[0]}


@pytest.mark.parametrize("codes", [True, False])
def test_the_sizes_reach_their_forms(codes):
    for size, (form, chunks) in SPLITS.items():
        assert chosen(*size, codes) == ([(form,)], chunks), size
    for (m, n, are_codes), form in LARGEST.items():
        found, chunks = chosen(m, n, LONG, are_codes, "float32")
        assert chunks == 1 and {f[-1] for f in found} == {form}, (m, n)
    assert {s[0] for s in SPLITS.values()} == set(SPLIT_FORMS) and set(LARGEST.values()) == set(FORMS)


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", SPLITS)
@pytest.mark.parametrize("codes", [True, False])
def test_chunks_of_k(device, m, n, k, codes):
    at = list(SPLITS).index((m, n, k))
    check_product(m, n, k, (F32, F16, BF16)[at % 3], device, codes, (None, "f32", "same")[at // 2 % 3])
    check_product(m, n, k, (F32, F16, BF16)[(at + 1) % 3], device, codes, None, seed=1, pads=(5, 0, 3) if codes else (0, 16, 0), offsets=(0, 0, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, codes", LARGEST)
def test_the_largest_sums_of_whole_k(device, m, n, codes):
    """Rows and channels of one value each, so that a sum is K times two codes: up to 131056 x 2^14 and down to 131056 x -127 x 128, in one
    accumulator."""

    row = torch.tensor([-128, 127, -127, 3, 126, -128, 1], device=device).repeat(m // 7 + 1)[:m]
    channel = torch.tensor([-128, -127, 127, 5, -128], device=device).repeat(n // 5 + 1)[:n]
    weight = channel.to(torch.int8)[:, None].expand(n, LONG).contiguous()
    w_scale = torch.linspace(0.001, 0.002, n, device=device)
    out = torch.empty(m, n, device=device)
    if codes:
        x_scale = torch.linspace(0.01, 0.02, m, device=device)
        native.int8_matmul(out, row.to(torch.int8)[:, None].expand(m, LONG).contiguous(), x_scale, weight, w_scale)
    else:
        row = torch.where(row < 0, -127, 127)  # the codes of rows of one value
        size = torch.linspace(0.5, 3.0, m, device=device)
        x_scale = size * torch.tensor(1 / 127, device=device)
        native.int8_matmul(out, (size * row.sign())[:, None].expand(m, LONG).contiguous(), None, weight, w_scale)
    part = (LONG * row[:, None] * channel).double() * x_scale.double()[:, None] * w_scale.double()
    error = (out.double() - part).abs()  # two products and the sum's rounding to 32 bits, and the result's own
    assert (error <= (3.01 * STEP + STEP + 1.01 * HALF[F32]) * part.abs()).all()
