"""Plain 64-bit forms of the serving operators (numpy, on the CPU), their error bounds, and input makers."""

from __future__ import annotations

import numpy as np
import torch

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
#: half a step of a type, relative to the value
HALF = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def f64(t) -> np.ndarray:
    return t.detach().cpu().to(torch.float64).numpy()


def quantised(x: torch.Tensor, dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """The documented 8-bit codes and scales of rows, in 32-bit steps on the CPU."""

    x = x.cpu().float()
    scale = x.abs().amax(-1) * torch.tensor(1.0 / LARGEST[dtype], dtype=torch.float32)
    code = torch.where((scale > 0)[..., None], x / scale[..., None], torch.zeros_like(x))
    code = code.clamp(-LARGEST[dtype], LARGEST[dtype])
    return (code.round() if dtype == torch.int8 else code).to(dtype), scale


def cache_values(cache, scale) -> np.ndarray:
    """[pages, heads, page_size, D] in 64 bits."""

    values = f64(cache)
    return values if scale is None else values * f64(scale)[..., None]


def make_cache(pages, heads, page_size, d, dtype, gen, model=torch.float32, scale_spread=0.5):
    """(cache, scales or None) on the CPU, rows of unequal size."""

    x = torch.randn(pages, heads, page_size, d, generator=gen)
    x = x * torch.exp(scale_spread * torch.randn(pages, heads, page_size, 1, generator=gen))
    if dtype in LARGEST:
        return quantised(x.to(model), dtype)
    return x.to(dtype), None


def page_table(lengths, page_size, pages, gen, columns=None):
    """Distinct pages in random order for sequences of these lengths; -1 past their last page."""

    need = [-(-n // page_size) for n in lengths]
    columns = max([1, *need]) if columns is None else columns
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    table, at = torch.full((len(lengths), columns), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n]
        at += n
    assert at <= pages
    return table


def tree_mask(parents: list[list[int]], words: int) -> torch.Tensor:
    """Bit rows of trees given as each token's parent (-1: the context alone)."""

    rows = []
    for tree in parents:
        seen: list[int] = []
        for j, p in enumerate(tree):
            assert p < j
            seen.append((seen[p] if p >= 0 else 0) | 1 << j)
        rows += [[(s >> 64 * w) & (2**64 - 1) for w in range(words)] for s in seen]
    return torch.from_numpy(np.array(rows, dtype=np.uint64).reshape(len(rows), words).view(np.int64).copy())


def tree_oracle(q, k_cache, v_cache, k_scale, v_scale, table, context, starts, mask, scale, out):
    """(expected, allowed error) in 64 bits; rows of no request keep `out`'s values with no error allowed.

    The error allowed, from the inputs alone (u: half a step of the output's type, p: of the type the
    weights are rounded to for the product with V, at most the same):
      - the output's rounding: u |O|, and 2^-25 in fp16, whose steps stay 2^-24 below 2^-14 (one such
        output: 2.70e-8 off at a value of about 1e-5, where u |O| and the rest come to 1.79e-8);
      - weights rounded one by one, the sum of weights over rounded or unrounded ones:
        p sum_j w_j (|V_j| + |O|);
      - a score off by e_j moves O by at most max_j e_j sum_j w_j |V_j - O|, with
        e_j = 2 (D + 4) 2^-24 |scale| |q||k_j| (a sum of D products in any order, the products with a
        key's scale and the call's), plus the argument of the exponential, |s_j - max| 2^-23, and 2^-22 for
        the exponential itself;
      - sums over n keys in any order and their joining: (n + 32) 2^-24 sum_j w_j (|V_j| + |O|).
    A weight is at least the type's least subnormal's half off (2^-25 for fp16 weights whose largest is 1 or more). Of a cache with
    scales what is rounded is 2^(s_j + log2 c_j - max_i(s_i + log2 c_i)), c_j key j's value scale, against a sum of
    2^(s_j - max_i(s_i + log2 c_i)): 2^-25 there is 2^-25 2^(max(s_i + log2 c_i) - max s_i) <= 2^-25 max c_i of a sum whose largest
    term is 1, for each code: 2^-25 max c sum_j |code_j|, which is more than 2^-25 sum_j c_j |code_j| where scales differ (one
    output of 16384: 2.92e-7 off, 2.55e-7 by the latter and all other terms). A weight of up to
    2^-25 so may round to 0, and 0 times an infinity is NaN by arithmetic: where an infinite value has such a weight (against
    the row's largest; e^-745 in 64 bits, where the oracle's own is 0), an infinite result may be NaN (allowed: infinity)."""

    u = HALF[q.dtype]
    keys, values = cache_values(k_cache, k_scale), cache_values(v_cache, v_scale)
    value_codes, value_scales = f64(v_cache), None if v_scale is None else f64(v_scale)
    pages, heads, page_size, d = keys.shape
    qs, expected = f64(q), f64(out).copy()
    allowed = np.zeros_like(expected)
    group = q.shape[1] // heads
    tiny = 2.0**-25 if q.dtype == torch.float16 else 0.0
    bits = None if mask is None else mask.cpu().numpy().view(np.uint64)
    for b in range(len(context)):
        c, n = int(context[b]), int(starts[b + 1]) - int(starts[b])
        reach = table.shape[1] * page_size
        pos = np.arange(min(c + n, reach))
        at = table.cpu().numpy()[b, pos // page_size] if len(pos) else np.zeros(0, int)
        real = (at >= 0) & (at < pages)
        for j in range(n):
            t = int(starts[b]) + j
            seen = real.copy()
            for i in range(max(0, len(pos) - c)):
                hit = i <= j if bits is None else i // 64 < bits.shape[1] and bool(int(bits[t, i // 64]) >> (i % 64) & 1)
                seen[c + i] &= hit
            for h in range(q.shape[1]):
                if not seen.any():
                    expected[t, h], allowed[t, h] = 0.0, 0.0
                    continue
                kk = keys[at[seen], h // group, pos[seen] % page_size]
                vv = values[at[seen], h // group, pos[seen] % page_size]
                with np.errstate(all="ignore"):
                    s = scale * (kk @ qs[t, h])
                    top = max(s.max(), -2e38)
                    w = np.exp(s - top)
                    total = w.sum()
                    w = w / total if total != 0 else w
                    o = w @ vv
                    spread = w @ (np.abs(vv) + np.abs(o))
                    e = 2 * (d + 4) * 2.0**-24 * abs(scale) * (np.abs(kk) @ np.abs(qs[t, h])) + np.abs(s - top) * 2.0**-23 + 2.0**-22
                    expected[t, h] = o
                    small = (np.exp(s - top) <= 2 * tiny)[:, None] & np.isinf(vv)
                    lost = np.abs(vv).sum(0)
                    if v_scale is not None:
                        own = value_scales[at[seen], h // group, pos[seen] % page_size]
                        codes = np.abs(value_codes[at[seen], h // group, pos[seen] % page_size]).sum(0)
                        lost = np.maximum(lost, codes * np.abs(own).max())
                    allowed[t, h] = (u * np.abs(o) + (u + (len(s) + 32) * 2.0**-24) * spread + e.max() * spread
                                     + tiny * lost / max(total, 1.0) + tiny + 1e-30)
                    allowed[t, h][np.isinf(o)] = 0.0
                    allowed[t, h][np.isinf(o) & small.any(0)] = np.inf
    return expected, allowed


def assert_rows(got, expected, allowed, what=""):
    """Equal infinities and NaN, the rest within the bound."""

    got = f64(got)
    assert got.shape == expected.shape
    fine = np.isfinite(expected)
    either = np.isinf(expected) & np.isinf(allowed)  # an infinity or NaN
    assert not np.isfinite(got[either]).any(), what
    assert np.array_equal(np.isnan(got[~either]), np.isnan(expected[~either])), f"{what}: NaN in other places"
    infinite = np.isinf(expected) & ~either
    assert np.array_equal(got[infinite], expected[infinite]), what
    err = np.abs(got[fine] - expected[fine])
    bad = err > allowed[fine]
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.size} outside the bound; worst {err[bad].max():.3e} against "
                           f"{allowed[fine][bad][err[bad].argmax()]:.3e}")


def adapter_oracle(x, weight, bias, a, b, index, scale, roundings=2):
    """(expected, allowed error) in 64 bits. The error allowed (u: half a step of the type; matrix sums of n
    products in 32 bits in any order: n 2^-24 of the sum of magnitudes, at most):
      - `roundings` of the output, u each, of the output or of the projection without the adapter;
      - t = scale x A rounded to the type: u |t| |B|;
      - the three sums."""

    u = HALF[x.dtype]
    xs, ws, as_, bs = f64(x), f64(weight), f64(a), f64(b)
    base = xs @ ws + (0.0 if bias is None else f64(bias))
    k, rank = xs.shape[1], as_.shape[2]
    sums = (k + 2) * 2.0**-24 * (np.abs(xs) @ np.abs(ws) + (0.0 if bias is None else np.abs(f64(bias))))
    out, allowed = base.copy(), sums
    for l in range(as_.shape[0]):
        rows = np.nonzero(index.cpu().numpy() == l)[0]
        s = 1.0 if scale is None else float(scale[l])
        t = s * (xs[rows] @ as_[l])
        size = abs(s) * (np.abs(xs[rows]) @ np.abs(as_[l]))
        out[rows] += t @ bs[l]
        allowed[rows] += ((u + 2.0**-24) * np.abs(t) + (k + 2) * 2.0**-24 * size) @ np.abs(bs[l])
        allowed[rows] += (rank + 2) * 2.0**-24 * (size @ np.abs(bs[l]))
    allowed += u * np.abs(out) + (roundings - 1) * u * np.abs(base) + 1e-30
    if x.dtype == torch.float16:
        allowed += 2.0**-25 * roundings  # half a subnormal step
    return out, allowed * (1 + 2 * u)
