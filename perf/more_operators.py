"""More serving operators of this framework as they are measured: what a step runs between its tokens and its
attention, with projections in 8-bit integers. Pages and slots of the paged cache found on the GPU from the
requests' lengths, rows quantised, a matrix product in 8-bit integers with a scale for each token and channel,
norms of queries and keys for each head with the position rotation in the same pass.

listed() holds the named cases, draw() more of the same ranges. prepare() makes what a program holds
before a call, run() is one call: in plain torch where `own` is false, through
kernelcode_generate_amd.native where it is true. exact() is the same result in 64 bits.
"""

from __future__ import annotations

import functools
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "codes": 1}
TINY = 2.0 ** -149  # the least positive 32-bit value: scales above it divide
EPS = 1e-6
REACH = 32768  # positions of the rotation's table


def listed() -> list[dict]:
    return [
        # One decoding step of 256 requests of unequal length: a token each, on pages of 16 tokens. One request in
        # sixteen takes a new page; the step's pages go back as those of rejected drafts do.
        pages_case("pages_step", 256, 1, 8192, 16, 256, 1.0, 1),
        # Prompts come in for 24 requests, behind cached beginnings, in a batch padded to 16384 tokens; then they end.
        pages_case("pages_prompts", 24, 1100, 1000, 16, 16384, 1.0, 2),
        # The rows of one decoding step before a projection. The smallest call there is.
        rows_case("rows_bf16_step", "bf16", 16, 4096),
        # The rows of prompts, of odd number.
        rows_case("rows_f16_prompt", "f16", 4001, 4096),
        # One decoding step of 16 requests through a projection, rows quantised in the call: its weights are the
        # whole call.
        int8_case("int8_bf16_step", "bf16", "bf16", 16, 4096, 4096, "none"),
        # Drafted tokens and short prompts in one batch of no whole tile.
        int8_case("int8_bf16_batch", "bf16", "bf16", 300, 4096, 4096, "f32"),
        # Odd extents throughout, with a bias.
        int8_case("int8_f16_odd", "f16", "f16", 1000, 1023, 1501, "same"),
        # Prompts at the benchmark's headline extents, rows quantised in the call.
        int8_case("int8_bf16_4096", "bf16", "bf16", 4096, 4096, 4096, "none"),
        # Long prompts in a wide layer, of codes that are there already: the largest product.
        int8_case("int8_codes_8192", "codes", "bf16", 8192, 8192, 8192, "none"),
        # Queries and keys of one decoding step of 64 requests, views of a fused projection: 32 and 8 heads of 128.
        rotate_case("rotate_bf16_step", "bf16", 64, 32, 8, 128, 128, "halves", "same"),
        # Those of prompts of 8192 tokens, one in sixteen padding.
        rotate_case("rotate_bf16_prompt", "bf16", 8192, 32, 8, 128, 128, "halves", "f32"),
        # Heads of 80 of which 32 elements turn, neighbours as pairs, no norms, an odd number of tokens.
        rotate_case("rotate_f16_part", "f16", 777, 12, 12, 80, 32, "neighbours", "none"),
    ]


def pages_case(name, batch, new, context, page, tokens, spare, ragged) -> dict:
    """new: tokens of a request, context: cached ones, up to that many; tokens: rows of the batch; spare: free pages,
    of those that the call takes (below 1: some requests get none)."""
    return {"name": name, "op": "pages", "batch": batch, "new": new, "context": context, "page": page, "tokens": tokens,
            "spare": spare, "ragged": ragged}


def rows_case(name, dtype, rows, k) -> dict:
    return {"name": name, "op": "rows", "dtype": dtype, "rows": rows, "k": k}


def int8_case(name, x, dtype, rows, k, n, bias) -> dict:
    """x: codes with scales, or rows of the output's type that the call quantises."""
    return {"name": name, "op": "int8", "x": x, "dtype": dtype, "rows": rows, "k": k, "n": n, "bias": bias}


def rotate_case(name, dtype, tokens, heads_q, heads, d, turned, pairs, weights) -> dict:
    """turned: elements of a head that the rotation takes; weights: type of the norms' weights (none: no norms)."""
    return {"name": name, "op": "rotate", "dtype": dtype, "tokens": tokens, "heads_q": heads_q, "heads": heads, "d": d,
            "turned": turned, "pairs": pairs, "weights": weights}


def log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    while True:
        op = rng.choice(("pages", "rows", "int8", "int8", "int8", "rotate", "rotate"))
        case = {"pages": draw_pages, "rows": draw_rows, "int8": draw_int8, "rotate": draw_rotate}[op](rng)
        if case is not None:
            del case["name"]
            return case


def draw_pages(rng) -> dict | None:
    """Steps, drafts and prompts of up to 1024 requests and 16384 tokens; batches padded, or too short for all."""
    mode = rng.choice(("step", "drafts", "prompts"))
    new, batch = {"step": (1, log_int(rng, 1, 1024)), "drafts": (log_int(rng, 2, 64), log_int(rng, 1, 256)),
                  "prompts": (log_int(rng, 64, 4096), log_int(rng, 1, 32))}[mode]
    tokens = max(1, int(batch * new * rng.choice((0.5, 0.75, 1, 1, 1.5))))
    case = pages_case("", batch, new, log_int(rng, 1, 16384), rng.choice((16, 16, 32, 64, 1, 24)), tokens,
                      rng.choice((1.0, 1.0, 2.0, 0.5)), rng.randrange(1, 1 << 20))
    table = batch * (case["context"] + new) / case["page"]
    return case if tokens <= 16384 and table <= 2e6 else None


def draw_rows(rng) -> dict | None:
    """From one row to prompts of 8192, of any length from 64 to 16384."""
    k = log_int(rng, 64, 16384)
    case = rows_case("", rng.choice(("bf16", "bf16", "f16", "f32")), log_int(rng, 1, 8192), k if rng.random() < 0.3 else k // 16 * 16)
    return case if work(case)["bytes"] <= 2e8 else None


def draw_int8(rng) -> dict | None:
    """Rows from one token to a batch of prompts; the extents of layers, mostly multiples of 16."""
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    k, n = log_int(rng, 64, 16384), log_int(rng, 64, 16384)
    if rng.random() < 0.75:
        k, n = max(k // 16, 1) * 16, max(n // 16, 1) * 16
    case = int8_case("", rng.choice(("codes", dtype)), dtype, log_int(rng, 1, 8192), k, n, rng.choice(("none", "f32", "same")))
    needs = work(case)
    return case if needs["flops"] <= 3e11 and needs["bytes"] <= 4e8 else None


def draw_rotate(rng) -> dict | None:
    """From one token to prompts of 8192, one to eight query heads per key head, heads turned whole or in part."""
    d, heads = rng.choice((64, 128, 128, 80, 96, 256, 72)), rng.choice((1, 2, 4, 8, 12, 16))
    case = rotate_case("", rng.choice(("bf16", "bf16", "f16", "f32")), log_int(rng, 1, 8192), heads * rng.choice((1, 2, 4, 8)), heads,
                       d, rng.choice((d, d, d // 2, d // 4 // 2 * 2)), rng.choice(("halves", "halves", "neighbours")),
                       rng.choice(("same", "f32", "none")))
    return case if work(case)["bytes"] <= 5e8 else None


def lengths(case) -> tuple[list[int], list[int]]:
    """(cached tokens, new tokens) of each request; one in twelve has no new ones."""
    rng = random.Random(case["ragged"])
    cached = [rng.randint(0, case["context"]) for _ in range(case["batch"])]
    new = [0 if rng.random() < 1 / 12 else rng.randint((case["new"] + 1) // 2, case["new"]) for _ in range(case["batch"])]
    return cached, new


def fitting(case) -> tuple[list[int], list[int], list[int]]:
    """(cached tokens, new tokens that the batch has rows for, first row) of each request."""
    cached, new = lengths(case)
    kept, starts, at = [], [], 0
    for n in new:
        starts.append(at)
        kept.append(min(n, case["tokens"] - at))
        at += kept[-1]
    return cached, kept, starts


def page_count(case, tokens: int) -> int:
    return -(-tokens // case["page"])


def quantised(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows as 8-bit integers and their 32-bit scales."""
    x = x.float()
    scale = x.abs().amax(-1) * torch.tensor(1.0 / 127.0, dtype=torch.float32, device=x.device)
    whole = torch.where((scale >= TINY)[:, None], x / scale[:, None], torch.zeros_like(x))
    return whole.clamp(-127, 127).round().to(torch.int8), scale


def generator(seed: int) -> torch.Generator:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    return gen


def inputs(case, seed: int) -> dict:
    return {"pages": pages_inputs, "rows": rows_inputs, "int8": int8_inputs, "rotate": rotate_inputs}[case["op"]](case, generator(seed))


def pages_inputs(case, gen) -> dict:
    cached, new = lengths(case)
    _, kept, _ = fitting(case)
    batch, width = case["batch"], max(1, page_count(case, case["context"] + case["new"]))
    held = torch.tensor([page_count(case, c) for c in cached])
    wanted = sum(page_count(case, c + n) - page_count(case, c) for c, n in zip(cached, kept))
    used, free = int(held.sum()), int(case["spare"] * wanted) + (8 if case["spare"] >= 1 else 0)
    pages = torch.randperm(used + free, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    there = (torch.arange(width) < held[:, None]).cuda()
    table[there] = pages[:used]
    stack = torch.full((used + free,), -1, dtype=torch.int32, device="cuda")
    stack[:free] = pages[used:]

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    return {"table": table, "free": stack, "count": whole([free]), "cached": whole(cached), "new": whole(new),
            "after": whole([c + n for c, n in zip(cached, kept)])}


def activations(rows: int, k: int, dtype, gen) -> torch.Tensor:
    """Rows of unequal size, with a few channels that are larger than the rest."""
    x = torch.randn((rows, k), generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device="cuda"))
    x *= torch.where(torch.rand((1, k), generator=gen, device="cuda") < 0.005, 8.0, 1.0)
    return x.to(dtype)


def rows_inputs(case, gen) -> dict:
    return {"x": activations(case["rows"], case["k"], DTYPES[case["dtype"]], gen)}


def int8_inputs(case, gen) -> dict:
    m, k, n = case["rows"], case["k"], case["n"]
    x, x_scale = activations(m, k, DTYPES[case["dtype"]], gen), None
    if case["x"] == "codes":
        x, x_scale = quantised(x)
    weight, w_scale = quantised(torch.randn((n, k), generator=gen, device="cuda") * 0.02)
    bias = None
    if case["bias"] != "none":
        bias = (torch.randn(n, generator=gen, device="cuda") * 0.02).to(DTYPES["f32" if case["bias"] == "f32" else case["dtype"]])
    return {"x": x, "x_scale": x_scale, "weight": weight, "w_scale": w_scale, "bias": bias}


def rotate_inputs(case, gen) -> dict:
    t, heads_q, heads, d, turned, dtype = (case[x] for x in ("tokens", "heads_q", "heads", "d", "turned", "dtype"))
    fused = torch.randn((t, heads_q + 2 * heads, d), generator=gen, device="cuda")  # as one projection gives them
    fused = (fused * torch.exp(0.5 * torch.randn((t, 1, 1), generator=gen, device="cuda"))).to(DTYPES[dtype])
    rate = 10000.0 ** (-torch.arange(turned // 2, dtype=torch.float64, device="cuda") / max(turned // 2, 1))
    angle = torch.arange(REACH, dtype=torch.float64, device="cuda")[:, None] * rate
    positions = torch.randint(0, REACH, (t,), generator=gen, device="cuda", dtype=torch.int32)
    positions = positions if t <= 256 else (positions[:1] % (REACH - t) + torch.arange(t, device="cuda")).to(torch.int32)  # a prompt
    positions[t - t // 16 :] = -1  # padding of the batch: left as it is
    weights = [None, None]
    if case["weights"] != "none":
        kind = DTYPES["f32" if case["weights"] == "f32" else dtype]
        weights = [(1 + 0.3 * torch.randn(d, generator=gen, device="cuda")).to(kind) for _ in range(2)]
    return {"q": fused[:, :heads_q], "k": fused[:, heads_q : heads_q + heads], "weights": weights, "positions": positions,
            "cos": torch.cos(angle).float(), "sin": torch.sin(angle).float()}


def prepare(case, seed):
    state = inputs(case, seed)
    state["case"] = case

    def buffer(*shape, dtype):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    if case["op"] == "pages":
        state["slots"] = buffer(case["tokens"], dtype=torch.int64)
        state["positions"] = buffer(case["tokens"], dtype=torch.int32)
        state["starts"] = buffer(case["batch"] + 1, dtype=torch.int32)
    elif case["op"] == "rows":
        state["codes"] = buffer(case["rows"], case["k"], dtype=torch.int8)
        state["scale"] = buffer(case["rows"], dtype=torch.float32)
    elif case["op"] == "int8":
        state["out"] = buffer(case["rows"], case["n"], dtype=DTYPES[case["dtype"]])
    else:
        for x in ("q", "k"):
            state[x + "_out"] = buffer(*state[x].shape, dtype=state[x].dtype)
    return state


@functools.lru_cache(None)
def native():
    """The framework's entries, enqueueing on torch's stream as a program does that goes on with torch."""
    from kernelcode_generate_amd import native as entries

    entries.set_launch_mode(False, torch.cuda.current_stream().cuda_stream)
    return entries


def run(state):
    return {"pages": run_pages, "rows": run_rows, "int8": run_int8, "rotate": run_rotate}[state["case"]["op"]](state)


def run_pages(s):
    """Pages and slots of the new tokens, then back to the cached ones (drafts rejected, requests ended), which
    leaves pages and stack as they were."""
    table, free, count, page = s["table"], s["free"], s["count"], s["case"]["page"]
    if own:
        entries = native()
        entries.kv_cache_assign(s["slots"], s["positions"], s["starts"], table, free, count, s["cached"], s["new"], page)
        entries.kv_cache_release(table, free, count, s["cached"], s["after"], page)
        return [s["slots"], s["positions"], s["starts"], table, free, count]
    cached, total = s["cached"].long(), s["case"]["tokens"]
    ends = torch.cumsum(s["new"].long().clamp(min=0), 0).clamp(max=total)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    width = table.shape[1]
    held = ((cached + page - 1) // page).clamp(max=width)
    need = ((cached + starts[1:] - starts[:-1] + page - 1) // page).clamp(max=width)
    taken = torch.cumsum(need - held, 0)
    column = torch.arange(width, device="cuda")
    place = (taken - (need - held))[:, None] + column - held[:, None]  # of a new page among all of them
    fresh = (column >= held[:, None]) & (column < need[:, None])
    picked = torch.where(place < count, free[(count - 1 - place).clamp(0, free.shape[0] - 1).long()], -1)
    table.copy_(torch.where(fresh, picked, table))
    count.sub_(torch.minimum(taken[-1:], count.long()).to(torch.int32))
    row = torch.arange(total, device="cuda")
    owner = (torch.searchsorted(starts, row, right=True) - 1).clamp(max=held.shape[0] - 1)
    real = row < starts[-1]
    position = cached[owner] + row - starts[owner]
    at = position // page
    own_page = torch.where(at < width, table[owner, at.clamp(max=width - 1)], -1).long()
    slots = torch.where(real & (own_page >= 0), own_page * page + position % page, -1)
    positions = torch.where(real, position, -1).to(torch.int32)
    # back: the entries of these pages in order, the first of them on top
    last = ((s["after"].long() + page - 1) // page).clamp(max=width)
    gone = (column >= held[:, None]) & (column < last[:, None]) & (table >= 0)
    order = torch.cumsum(gone.flatten().long(), 0)
    back = order[-1:]
    spot = torch.where(gone.flatten(), count + back - order, free.shape[0])
    longer = torch.cat([free, free.new_zeros(1)])
    longer[spot] = table.flatten()
    free.copy_(longer[:-1])
    table.masked_fill_(gone, -1)
    count.add_(back.to(torch.int32))
    return [slots, positions, starts.to(torch.int32), table, free, count]


def run_rows(s):
    if own:
        native().quantize_rows(s["codes"], s["scale"], s["x"])
        return [s["codes"], s["scale"]]
    return list(quantised(s["x"]))


def run_int8(s):
    if own:
        native().int8_matmul(s["out"], s["x"], s["x_scale"], s["weight"], s["w_scale"], s["bias"])
        return s["out"]
    codes, scale = quantised(s["x"]) if s["x_scale"] is None else (s["x"], s["x_scale"])
    out = codes.float() @ s["weight"].float().t()
    out = out * scale[:, None] * s["w_scale"]
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return out.to(s["out"].dtype)


def run_rotate(s):
    neighbours = s["case"]["pairs"] == "neighbours"
    if own:
        native().head_norm_rotate(s["q_out"], s["k_out"], s["q"], s["k"], *s["weights"], s["cos"], s["sin"], s["positions"],
                                  EPS, neighbours)
    else:
        there = (s["positions"] >= 0)[:, None, None]
        at = s["positions"].clamp(min=0).long()
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        for x, weight in zip(("q", "k"), s["weights"]):
            rows = s[x].float()
            if weight is not None:
                rows = rows * torch.rsqrt((rows * rows).mean(-1, keepdim=True) + EPS) * weight.float()
            rows = plain_turned(rows, cos, sin, neighbours)
            s[x + "_out"].copy_(torch.where(there, rows.to(s[x].dtype), s[x + "_out"]))
    return [s["q_out"], s["k_out"]]


def plain_turned(rows, cos, sin, neighbours):
    half = cos.shape[-1]
    turned, rest = rows[..., : 2 * half], rows[..., 2 * half :]
    a, b = (turned[..., ::2], turned[..., 1::2]) if neighbours else (turned[..., :half], turned[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if neighbours else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def work(case):
    if case["op"] == "pages":
        cached, kept, _ = fitting(case)
        pages = sum(page_count(case, c + n) - page_count(case, c) for c, n in zip(cached, kept))
        # lengths, starts, slots and positions, a page of each request looked up; of each new page both lists and back
        return {"bytes": 20.0 * case["batch"] + 12.0 * case["tokens"] + 32.0 * pages, "flops": 0.0}
    size = BYTES[case["dtype"]]
    if case["op"] == "rows":
        return {"bytes": float(case["rows"] * (case["k"] * (size + 1) + 4)), "flops": 0.0}
    if case["op"] == "int8":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": float(m * k * BYTES[case["x"]] + n * k + m * n * size + 4 * n), "flops": 2.0 * m * k * n}
    t = case["tokens"] - case["tokens"] // 16
    return {"bytes": float(t * (2 * (case["heads_q"] + case["heads"]) * case["d"] * size + 4 * case["turned"] + 4)), "flops": 0.0}


def exact(case, seed):
    """run()'s outputs from the definition: whole numbers request by request, the others in 64 bits."""
    s = inputs(case, seed)
    return {"pages": exact_pages, "rows": exact_rows, "int8": exact_int8, "rotate": exact_rotate}[case["op"]](case, s)


def exact_pages(case, s):
    cached, kept, starts = fitting(case)
    page, table, free = case["page"], s["table"].tolist(), s["free"].tolist()
    stack = free[: int(s["count"])]
    slots, positions = [-1] * case["tokens"], [-1] * case["tokens"]
    for b, (c, n) in enumerate(zip(cached, kept)):
        pages = table[b]
        for p in range(page_count(case, c), page_count(case, c + n)):
            pages[p] = stack.pop() if stack else -1
        for i in range(n):
            positions[starts[b] + i] = c + i
            own_page = pages[(c + i) // page]
            slots[starts[b] + i] = own_page * page + (c + i) % page if own_page >= 0 else -1
    # what goes back restores the stack and the table
    whole = [(slots, torch.int64), (positions, torch.int32), (starts + [starts[-1] + kept[-1]], torch.int32)]
    return [torch.tensor(x, dtype=t, device="cuda") for x, t in whole] + [s["table"], s["free"], s["count"]]


def exact_codes(x):
    """The whole numbers nearest to the 32-bit quotients by the 32-bit scale, ties to even."""
    top = x.double().abs().amax(-1)
    scale = (top * float(torch.tensor(1.0 / 127.0, dtype=torch.float32))).float().double()
    quotient = torch.nan_to_num(x.double() / scale[:, None], posinf=0.0, neginf=0.0).float().double()
    return torch.round(quotient).clamp(-127, 127), scale


def exact_rows(case, s):
    codes, scale = exact_codes(s["x"])
    return [codes.to(torch.int8), scale]


def exact_int8(case, s):
    codes, scale = exact_codes(s["x"]) if s["x_scale"] is None else (s["x"].double(), s["x_scale"].double())
    out = torch.mm(codes, s["weight"].double().t().contiguous())
    out *= scale[:, None]
    out *= s["w_scale"].double()
    return out if s["bias"] is None else out + s["bias"].double()


def exact_rotate(case, s):
    there = (s["positions"] >= 0).nonzero().flatten()
    at, half = s["positions"][there].long(), case["turned"] // 2
    cos, sin = s["cos"].double()[at], s["sin"].double()[at]
    step, other = (2, 1) if case["pairs"] == "neighbours" else (1, half)  # from pair to pair, and within one
    outs = []
    for x, weight in zip(("q", "k"), s["weights"]):
        out = torch.zeros(s[x].shape, dtype=torch.float64, device="cuda")
        for h in range(out.shape[1]):
            y = s[x][there, h].double()
            if weight is not None:
                y = y / torch.sqrt(y.pow(2).mean(1, keepdim=True) + EPS) * weight.double()
            first = torch.arange(half, device="cuda") * step
            a, b = y[:, first], y[:, first + other]
            y[:, first], y[:, first + other] = a * cos - b * sin, a * sin + b * cos
            out[there, h] = y
        outs.append(out)
    return outs
