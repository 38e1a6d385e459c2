"""Plain forms, in whole numbers and 64 bits on the CPU, of the entries that a serving step runs between its tokens and its
attention, with their error bounds."""

from __future__ import annotations

import numpy as np
import torch

from tests.serving_util import HALF, f64

STEP = 2.0**-24  # half a step of 32 bits, relative


def ceil_pages(tokens: int, page_size: int, per: int) -> int:
    return min(-(-max(tokens, 0) // page_size), per)


def assign_oracle(table, free, count, context, added, page_size, tokens):
    """(slots, positions, starts, table, count) of lists; the tables as lists of lists."""

    table, left = [list(row) for row in table], max(0, min(count, len(free)))
    per = len(table[0]) if table else 0
    slots, positions, starts = [-1] * tokens, [-1] * tokens, [0]
    for b, (c, n) in enumerate(zip(context, added)):
        c, n = max(c, 0), min(max(n, 0), tokens - starts[-1])
        for p in range(ceil_pages(c, page_size, per), ceil_pages(c + n, page_size, per)):
            table[b][p] = free[left - 1] if left else -1
            left -= left > 0
        for i in range(n):
            pos, row = c + i, starts[-1] + i
            positions[row] = pos
            page = table[b][pos // page_size] if pos // page_size < per else -1
            slots[row] = page * page_size + pos % page_size if page >= 0 else -1
        starts.append(starts[-1] + n)
    return slots, positions, starts, table, left


def release_oracle(table, free, count, keep, held, page_size):
    """(table, free, count) of lists."""

    table, free, count = [list(row) for row in table], list(free), max(0, min(count, len(free)))
    per = len(table[0]) if table else 0
    pages = []
    for b, (k, h) in enumerate(zip(keep, held)):
        for p in range(ceil_pages(k, page_size, per), ceil_pages(h, page_size, per)):
            if table[b][p] >= 0:
                pages.append(table[b][p])
            table[b][p] = -1
    for i, page in enumerate(pages):
        spot = count + len(pages) - 1 - i
        if spot < len(free):
            free[spot] = page
    return table, free, min(count + len(pages), len(free))


def codes_oracle(x) -> tuple[np.ndarray, np.ndarray]:
    """Codes (int64) and 32-bit scales of rows, in the documented 32-bit steps."""

    x = x.detach().cpu().to(torch.float32).numpy()
    with np.errstate(all="ignore"):
        top = np.abs(x).max(1, initial=0.0)  # (a NaN stays)
        scale = (top * np.float32(1.0 / 127.0)).astype(np.float32)
        fine = np.isfinite(scale) & (scale > 0)
        code = np.zeros(x.shape)
        code[fine] = np.clip(np.rint((x[fine] / scale[fine, None]).astype(np.float32)), -127, 127)
    return code.astype(np.int64), scale


def int8_oracle(codes, x_scale, weight, w_scale, bias, dtype):
    """(expected, allowed error). The sum is exact in whole numbers; as a 32-bit float, its two products with the
    scales (three roundings, and half a least step of 32 bits, 2^-150, times what follows), the bias added (one, of the
    result), the output's own (and 2^-25 in fp16, half a subnormal step)."""

    sums = (torch.from_numpy(np.ascontiguousarray(codes)).double() @ weight.cpu().double().t()).numpy()  # below 2^53: exact
    assert np.abs(sums).max(initial=0) < 2**31
    ws = f64(w_scale)
    with np.errstate(all="ignore"):
        part = sums * x_scale.astype(np.float64)[:, None] * ws
        out = part if bias is None else part + f64(bias)
        allowed = 3.01 * STEP * np.abs(part) + (STEP + HALF[dtype] * 1.01) * np.abs(out) + 2.0**-149 * (1 + np.abs(ws))
    if dtype == torch.float16:
        allowed = allowed + 2.0**-25
    return out, allowed


def head_norm_oracle(x, weight, cos, sin, positions, eps, neighbours, out):
    """(expected, allowed error) of one side; tokens outside the table keep `out`'s values with no error allowed.

    The sum of D squares in any order is off by at most (D + 1) STEP of itself, its mean and eps by two roundings more, the inverse
    root by half of that and one step (two STEP) of its own: e = ((D + 3) / 2 + 2) STEP; products with it and the weight: 2 STEP.
    A turned element p cos - q sin: each product off by that and one rounding, the sum by one. Then the output's rounding."""

    xs, expected = f64(x), f64(out).copy()
    allowed, d, half = np.zeros_like(expected), x.shape[2], cos.shape[1]
    c, s, at = f64(cos), f64(sin), positions.cpu().numpy().astype(np.int64)
    u, tiny = HALF[x.dtype] * 1.01, 2.0**-25 if x.dtype == torch.float16 else 2.0**-140
    first = np.arange(half) * (2 if neighbours else 1)
    second = first + (1 if neighbours else half)
    for t in range(x.shape[0]):
        if not 0 <= at[t] < c.shape[0]:
            continue
        y, e = xs[t].copy(), 0.0
        if weight is not None:
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * f64(weight)
            e = ((d + 3) / 2 + 4) * STEP
        a, b = y[:, first], y[:, second]
        cc, ss = c[at[t]], s[at[t]]
        size = np.abs(y)
        turned = y.copy()
        turned[:, first], turned[:, second] = a * cc - b * ss, b * cc + a * ss
        size[:, first], size[:, second] = np.abs(a * cc) + np.abs(b * ss), np.abs(b * cc) + np.abs(a * ss)
        expected[t], allowed[t] = turned, (e + 2.1 * STEP) * size + u * np.abs(turned) + tiny
    return expected, allowed


def assert_close(got, expected, allowed, what=""):
    """Equal infinities and NaN, the rest within the bound."""

    got = f64(got)
    assert got.shape == expected.shape, what
    fine = np.isfinite(expected)
    assert np.array_equal(np.isnan(got), np.isnan(expected)), f"{what}: NaN in other places"
    infinite = np.isinf(expected)
    assert np.array_equal(got[infinite], expected[infinite]), what
    err = np.abs(got[fine] - expected[fine])
    bad = ~(err <= allowed[fine])
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.size} outside the bound; worst {err[bad].max():.3e} against "
                           f"{allowed[fine][bad][err[bad].argmax()]:.3e}")
