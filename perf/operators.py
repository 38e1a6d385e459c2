"""The serving operators of this framework as they are measured: a cache of keys and values written
and read back (in 16 bits, or in 8 bits with a scale per token and head), attention of tree-drafted
tokens over that cache, and a projection with the low-rank adapters of many requests beside it.

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

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8,
          "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "int8": 1, "e4m3": 1}
LARGEST = {"int8": 127.0, "e4m3": 448.0}  # of a quantised value; a row's scale is its largest magnitude over this
TINY = 2.0 ** -149  # the least positive 32-bit value: scales above it divide


def listed() -> list[dict]:
    return [
        # One decoding step of 64 sequences writes its keys and values: 8 heads of 128, pages of
        # 16 tokens, 8-bit floats. The smallest call there is.
        store_case("store_e4m3_step", "bf16", "e4m3", 64, 8, 128, 16),
        # A prompt of odd length goes to the cache as integers, pages of 64 tokens.
        store_case("store_int8_prompt", "f16", "int8", 4001, 8, 128, 64),
        # A short cache read back for an attention over dense tensors: 12 heads of 64.
        load_case("load_int8_short", "f16", "int8", 1, 12, 64, 16, 777, 0),
        # Four sequences of unequal length read back.
        load_case("load_e4m3_ragged", "bf16", "e4m3", 4, 8, 128, 16, 8192, 1),
        # One decoding step (a tree of one token) of 16 sequences of unequal length, four query heads
        # to a key head.
        tree_case("tree_bf16_step", "bf16", "bf16", 16, 8, 4, 128, 16, 1, "chain", 4096, 2),
        # Trees of 16 drafted tokens over an 8-bit cache.
        tree_case("tree_e4m3_drafts", "bf16", "e4m3", 8, 8, 4, 128, 64, 16, "tree", 8192, 3),
        # Odd trees, heads of 64 with keys of their own, integer cache, short contexts.
        tree_case("tree_int8_odd", "f16", "int8", 5, 12, 1, 64, 16, 25, "tree", 1000, 4),
        # One sequence with a long context: its keys are the whole call.
        tree_case("tree_bf16_long", "bf16", "bf16", 1, 8, 4, 128, 64, 1, "chain", 65536, 0),
        # Pieces of two prompts after 4096 cached tokens: matrix products, not bytes.
        tree_case("tree_bf16_prompt", "bf16", "bf16", 2, 8, 4, 128, 16, 512, "chain", 4096, 0),
        # One decoding step of 16 requests, each row with an adapter of its own out of 32.
        adapter_case("adapter_bf16_step", "bf16", 16, 4096, 4096, 32, 16, "mixed", "f32"),
        # Drafted tokens of many requests in one batch, rank 64, rows of one adapter apart.
        adapter_case("adapter_f16_mixed", "f16", 200, 2048, 2048, 16, 64, "mixed", "same"),
        # Prompts of several requests in one projection: runs of rows share an adapter.
        adapter_case("adapter_bf16_prompts", "bf16", 4096, 4096, 4096, 8, 16, "runs", "none"),
    ]


def store_case(name, dtype, cache, tokens, heads, d, page) -> dict:
    return {"name": name, "op": "store", "dtype": dtype, "cache": cache, "tokens": tokens, "heads": heads, "d": d,
            "page": page}


def load_case(name, dtype, cache, batch, heads, d, page, longest, ragged) -> dict:
    return {"name": name, "op": "load", "dtype": dtype, "cache": cache, "batch": batch, "heads": heads, "d": d,
            "page": page, "longest": longest, "ragged": ragged}


def tree_case(name, dtype, cache, batch, heads, group, d, page, tokens, mask, context, ragged) -> dict:
    """tokens: drafted ones of a sequence (ragged: up to that many, and contexts up to `context`)."""
    return {"name": name, "op": "tree", "dtype": dtype, "cache": cache, "batch": batch, "heads": heads, "group": group,
            "d": d, "page": page, "tokens": tokens, "mask": mask, "context": context, "ragged": ragged}


def adapter_case(name, dtype, rows, k, n, adapters, rank, order, bias) -> dict:
    return {"name": name, "op": "adapter", "dtype": dtype, "rows": rows, "k": k, "n": n, "adapters": adapters,
            "rank": rank, "order": order, "bias": bias}


def log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    while True:
        op = rng.choice(("store", "load", "tree", "tree", "tree", "adapter", "adapter"))
        case = {"store": draw_store, "load": draw_load, "tree": draw_tree, "adapter": draw_adapter}[op](rng)
        if case is not None:
            del case["name"]
            return case


def draw_heads(rng) -> tuple[str, str, int, int, int]:
    dtype = rng.choice(("bf16", "bf16", "f16"))
    cache = rng.choice((dtype, "e4m3", "int8"))
    return dtype, cache, rng.choice((1, 2, 4, 8, 12, 16)), rng.choice((64, 128, 128, 80, 256)), rng.choice((16, 16, 32, 64, 256, 1, 24))


def draw_store(rng) -> dict | None:
    """From one token to prompts of 8192, any number of heads, head sizes 64 to 256."""
    dtype, cache, heads, d, page = draw_heads(rng)
    case = store_case("", dtype, cache, log_int(rng, 1, 8192), heads, d, page)
    return case if work(case)["bytes"] <= 1e8 else None


def draw_load(rng) -> dict | None:
    dtype, cache, heads, d, page = draw_heads(rng)
    case = load_case("", dtype, cache, log_int(rng, 1, 32), heads, d, page, log_int(rng, 1, 16384), rng.randrange(1 << 20))
    return case if work(case)["bytes"] <= 2e8 else None


def draw_tree(rng) -> dict | None:
    """Decoding steps, trees of up to 80 drafted tokens and pieces of prompts, over contexts of 1 to 65536
    tokens, one to eight query heads per key head."""
    dtype, cache, heads, d, page = draw_heads(rng)
    mode = rng.choice(("step", "step", "tree", "tree", "prompt"))
    tokens, batch = {"step": (1, log_int(rng, 1, 64)), "tree": (log_int(rng, 2, 80), log_int(rng, 1, 16)),
                     "prompt": (log_int(rng, 64, 512), log_int(rng, 1, 4))}[mode]
    context = log_int(rng, 1, 65536 if mode == "step" else 16384)
    case = tree_case("", dtype, cache, batch, heads, rng.choice((1, 2, 4, 8)), d, page, tokens,
                     "tree" if mode == "tree" else "chain", context, rng.choice((0, rng.randrange(1, 1 << 20))))
    needs = work(case)
    widest = batch * (context + tokens) * heads * max(d, case["group"] * tokens)
    return case if needs["flops"] <= 1e11 and needs["bytes"] <= 5e8 and widest <= 3e8 else None


def draw_adapter(rng) -> dict | None:
    """Rows from one decoding sequence to a batch of prompts, the extents of layers (multiples of 8)."""
    rows, k, n = log_int(rng, 1, 8192), log_int(rng, 256, 8192) // 8 * 8, log_int(rng, 256, 8192) // 8 * 8
    rank, adapters = rng.choice((8, 16, 16, 32, 64)), log_int(rng, 1, 64)
    case = adapter_case("", rng.choice(("bf16", "bf16", "f16")), rows, k, n, adapters, rank, rng.choice(("mixed", "runs")),
                        rng.choice(("none", "f32", "same")))
    fits = work(case)["flops"] <= 1.4e11 and adapters * rank <= 1024
    return case if fits and (case["order"] == "runs" or rows <= 1024) else None


def lengths(case) -> tuple[list[int], list[int]]:
    """(cached tokens, new tokens) of each sequence: all alike, or (ragged: the seed) unequal ones."""
    longest, tokens, batch = case.get("longest", case.get("context")), case.get("tokens", 0), case["batch"]
    if not case["ragged"]:
        return [longest] * batch, [tokens] * batch
    rng = random.Random(case["ragged"])
    cached = [rng.randint(longest // 8, longest) for _ in range(batch)]
    return cached, [rng.randint((tokens + 1) // 2, tokens) for _ in range(batch)]


def quantised(x: torch.Tensor, cache: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of the last axis as 8-bit values and their 32-bit scales."""
    x = x.float()
    scale = x.abs().amax(-1) * torch.tensor(1.0 / LARGEST[cache], dtype=torch.float32, device=x.device)
    whole = torch.where((scale >= TINY)[..., None], x / scale[..., None], torch.zeros_like(x))
    whole = whole.clamp(-LARGEST[cache], LARGEST[cache])
    return (whole.round() if cache == "int8" else whole).to(DTYPES[cache]), scale


def bits(x: torch.Tensor) -> torch.Tensor:
    """8-bit floats as bytes, which torch can index."""
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def inputs(case, seed: int) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    if case["op"] == "adapter":
        return adapter_inputs(case, seed, normal)
    heads, d, page, cache = case["heads"], case["d"], case["page"], case["cache"]
    if case["op"] == "store":
        t, pages = case["tokens"], -(-4 * case["tokens"] // case["page"])
        fused = normal(t, 2 * heads, d)  # as the rows of one projection hold them
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:t]
        slots[t // 2 : t // 2 + t // 16] = -1  # padding of the batch: not written
        state = {"k": fused[:, :heads], "v": fused[:, heads:], "slots": slots}
    else:
        cached, new = lengths(case)
        per = max(-(-(c + n) // page) for c, n in zip(cached, new))
        pages = case["batch"] * per
        table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).reshape(case["batch"], per)
        used = torch.tensor([-(-(c + n) // page) for c, n in zip(cached, new)], device="cuda")
        table[torch.arange(per, device="cuda") >= used[:, None]] = -1  # no page
        state = {"table": table, "lens": torch.tensor(cached, dtype=torch.int32, device="cuda"), "reach": max(
            c + n for c, n in zip(cached, new))}
        if case["op"] == "tree":
            state.update(tree_inputs(case, seed, new, normal))
    for name in ("k", "v"):
        values = normal(pages, heads, page, d)
        if name == "v":  # values of tokens differ in size
            values = values * torch.exp(0.5 * torch.randn((pages, heads, page, 1), generator=gen, device="cuda")).to(dtype)
        state[name + "_cache"], state[name + "_scale"] = quantised(values, cache) if cache in LARGEST else (values, None)
    return state


def tree_inputs(case, seed, new, normal) -> dict:
    starts, rng = [0], random.Random(seed)
    for n in new:
        starts.append(starts[-1] + n)
    mask = None
    if case["mask"] == "tree":
        words = -(-case["tokens"] // 64)
        rows = []
        for n in new:
            seen = []
            for j in range(n):  # each token hangs on an earlier one, or on the context
                parent = rng.randrange(-1, j)
                seen.append((seen[parent] if parent >= 0 else 0) | 1 << j)
            rows += [[(s >> 64 * w & (1 << 64) - 1) - ((s >> 64 * w + 63 & 1) << 64) for w in range(words)] for s in seen]
        mask = torch.tensor(rows, dtype=torch.int64, device="cuda").reshape(starts[-1], words)
    return {"q": normal(starts[-1], case["heads"] * case["group"], case["d"]), "mask": mask, "most": max(new),
            "starts": torch.tensor(starts, dtype=torch.int32, device="cuda")}


def adapter_inputs(case, seed, normal) -> dict:
    m, k, n, count, rank = (case[x] for x in ("rows", "k", "n", "adapters", "rank"))
    rng = random.Random(seed)
    if case["order"] == "mixed":
        index = [rng.randrange(-1, count) for _ in range(m)]
    else:  # prompts of unequal length
        index = []
        while len(index) < m:
            index += [rng.randrange(-1, count)] * rng.randint(1, max(1, m // 4))
        index = index[:m]
    bias = {"none": None, "f32": normal(n, scale=0.02).float(), "same": normal(n, scale=0.02)}[case["bias"]]
    return {"x": normal(m, k), "w": normal(k, n, scale=0.02), "bias": bias, "a": normal(count, k, rank, scale=k ** -0.5),
            "b": normal(count, rank, n, scale=0.1), "index": torch.tensor(index, dtype=torch.int32, device="cuda"),
            "scale": torch.tensor([rng.uniform(0.5, 2.0) for _ in range(count)], dtype=torch.float32, device="cuda")}


def prepare(case, seed):
    state = inputs(case, seed)
    state["case"], dtype = case, DTYPES[case["dtype"]]
    if case["op"] == "load":
        shape = (case["batch"], case["heads"], state["reach"], case["d"])
        state["k_out"], state["v_out"] = (torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(2))
    elif case["op"] == "tree":
        state["out"] = torch.empty_like(state["q"])
    elif case["op"] == "adapter":
        state["out"] = torch.empty(case["rows"], case["n"], dtype=dtype, device="cuda")
    return state


@functools.lru_cache(None)
def native():
    """The framework's entries, enqueueing on torch's stream as a program does that goes on with torch."""
    from kernelcode_generate_amd import native as entries

    entries.set_launch_mode(False, torch.cuda.current_stream().cuda_stream)
    return entries


def run(state):
    return {"store": run_store, "load": run_load, "tree": run_tree, "adapter": run_adapter}[state["case"]["op"]](state)


def run_store(s):
    if own:
        native().kv_cache_store(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["k"], s["v"], s["slots"])
    else:
        kept = s["slots"] >= 0
        at, page = s["slots"][kept], s["case"]["page"]
        plain_store(s["k_cache"], s["k_scale"], s["k"][kept], at, page, s["case"]["cache"])
        plain_store(s["v_cache"], s["v_scale"], s["v"][kept], at, page, s["case"]["cache"])
    return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]


def plain_store(cache, scales, rows, at, page, kind):
    if scales is not None:
        rows, scale = quantised(rows, kind)
        scales[at // page, :, at % page] = scale
    bits(cache)[at // page, :, at % page] = bits(rows)


def plain_rows(cache, scales, table, reach):
    """[B, tokens, heads, D] in 32 bits: the values that the pages of a table hold."""
    page = cache.shape[2]
    pos = torch.arange(reach, device=cache.device)
    at = table[:, pos // page].clamp(min=0).long()
    rows = bits(cache)[at, :, pos % page]
    rows = (rows.view(cache.dtype) if cache.dtype == torch.float8_e4m3fn else rows).float()
    return rows if scales is None else rows * scales[at, :, pos % page][..., None]


def run_load(s):
    if own:
        native().kv_cache_load(s["k_out"], s["v_out"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                               s["lens"])
    else:
        held = torch.arange(s["reach"], device="cuda") < s["lens"][:, None]
        for x in ("k", "v"):
            rows = plain_rows(s[x + "_cache"], s[x + "_scale"], s["table"], s["reach"]).transpose(1, 2)
            s[x + "_out"].copy_(torch.where(held[:, None, :, None], rows, s[x + "_out"].float()))
    return [s["k_out"], s["v_out"]]


def run_tree(s):
    if own:
        native().tree_attention(s["out"], s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                                s["lens"], s["starts"], s["mask"], 1.0 / math.sqrt(s["case"]["d"]))
        return s["out"]
    case, starts, reach, most = s["case"], s["starts"].long(), s["reach"], s["most"]
    heads, group, d, total = case["heads"], case["group"], case["d"], s["q"].shape[0]
    step = torch.arange(most, device="cuda")
    token = (starts[:-1, None] + step).clamp(max=total - 1)  # [B, most]
    count = (starts[1:] - starts[:-1])[:, None]
    q = s["q"].float()[token].reshape(-1, most, heads, group, d).permute(0, 2, 1, 3, 4).reshape(-1, heads, most * group, d)
    k = plain_rows(s["k_cache"], s["k_scale"], s["table"], reach).permute(0, 2, 3, 1).contiguous()
    v = plain_rows(s["v_cache"], s["v_scale"], s["table"], reach).permute(0, 2, 1, 3).contiguous()
    draft = torch.arange(reach, device="cuda") - s["lens"][:, None].long()  # [B, reach]: below 0 in the context
    if s["mask"] is None:
        seen = draft[:, None] <= step[None, :, None]
    else:
        word = (draft // 64).clamp(0, s["mask"].shape[1] - 1)[:, None].expand(-1, most, -1)
        seen = (s["mask"][token].gather(2, word) >> (draft % 64)[:, None] & 1).bool() | (draft < 0)[:, None]
    seen &= (draft < count)[:, None]
    seen = seen[:, None, :, None, :].expand(-1, heads, -1, group, -1).reshape(-1, heads, most * group, reach)
    score = torch.matmul(q, k) / math.sqrt(d)
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=TINY)
    o = o.reshape(-1, heads, most, group, d).permute(0, 2, 1, 3, 4).reshape(-1, most, heads * group, d)
    at = torch.arange(total, device="cuda")
    owner = torch.searchsorted(starts, at, right=True) - 1
    return o[owner, at - starts[owner]].to(DTYPES[case["dtype"]])


def run_adapter(s):
    if own:
        native().adapter_matmul(s["out"], s["x"], s["w"], s["bias"], s["a"], s["b"], s["index"], s["scale"])
        return s["out"]
    count, k, rank = s["a"].shape
    x = s["x"].float()
    out = x @ s["w"].float()
    if s["bias"] is not None:
        out += s["bias"].float()
    chosen = (s["index"][:, None] == torch.arange(count, device="cuda")) * s["scale"]
    low = (x @ s["a"].float().transpose(0, 1).reshape(k, count * rank)).reshape(-1, count, rank) * chosen[..., None]
    out += low.reshape(-1, count * rank) @ s["b"].float().reshape(count * rank, -1)
    return out.to(DTYPES[s["case"]["dtype"]])


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "adapter":
        m, k, n, rank = case["rows"], case["k"], case["n"], case["rank"]
        used = min(m, case["adapters"]) if case["order"] == "mixed" else 1  # adapters that are read at least
        return {"bytes": float((m * k + k * n + m * n + used * rank * (k + n)) * size),
                "flops": 2.0 * m * k * n + 2.0 * m * rank * (k + n)}
    row = case["heads"] * case["d"]  # of one token
    kept = row * BYTES[case["cache"]] + (4 * case["heads"] if case["cache"] in LARGEST else 0)
    if case["op"] == "store":
        t = case["tokens"]
        return {"bytes": float(2 * (t - t // 16) * (row * size + kept) + 8 * t), "flops": 0.0}
    cached, new = lengths(case)
    if case["op"] == "load":
        return {"bytes": float(2 * sum(cached) * (kept + row * size)), "flops": 0.0}
    chain = case["mask"] == "chain"
    pairs = sum(n * c + (n * (n + 1) // 2 if chain else n) for c, n in zip(cached, new))
    return {"bytes": float(2 * (sum(cached) + sum(new)) * kept + 2 * sum(new) * case["group"] * row * size),
            "flops": 4.0 * case["group"] * row * pairs}


def exact(case, seed):
    """run()'s outputs in float64: one sequence, head or adapter at a time."""
    s = inputs(case, seed)
    return {"store": exact_store, "load": exact_load, "tree": exact_tree, "adapter": exact_adapter}[case["op"]](case, s)


def held(s, x) -> torch.Tensor:
    """[pages, heads, page, D]: what a cache's values stand for."""
    values = s[x + "_cache"].double()
    return values if s[x + "_scale"] is None else values * s[x + "_scale"].double()[..., None]


def exact_store(case, s):
    caches, scales = [], []
    for x in ("k", "v"):
        cache, scale, rows = s[x + "_cache"].double(), s[x + "_scale"], s[x].double()
        scale = None if scale is None else scale.double()
        kept = torch.nonzero(s["slots"] >= 0).flatten()
        page, at = s["slots"][kept] // case["page"], s["slots"][kept] % case["page"]
        rows = rows[kept]
        if scale is not None:
            size = rows.abs().max(-1).values / LARGEST[case["cache"]]
            scale[page, :, at] = size
            rows = torch.nan_to_num(rows / size[..., None]).float().to(torch.float8_e4m3fn).double()
        cache[page, :, at] = rows
        caches.append(None if case["cache"] == "int8" else cache)  # whole numbers: equal or not
        scales.append(scale)
    return caches + scales


def exact_load(case, s):
    outs = []
    for x in ("k", "v"):
        values, out = held(s, x), torch.zeros(case["batch"], case["heads"], s["reach"], case["d"], dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            pages = s["table"][b, : -(-n // case["page"])].long()
            out[b, :, :n] = values[pages].transpose(0, 1).reshape(case["heads"], -1, case["d"])[:, :n]
        outs.append(out)
    return outs


def exact_tree(case, s):
    keys, values, group = held(s, "k"), held(s, "v"), case["group"]
    starts, out = s["starts"].tolist(), torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, context in enumerate(s["lens"].tolist()):
        first, n = starts[b], starts[b + 1] - starts[b]
        pages = s["table"][b, : -(-(context + n) // case["page"])].long()
        drafts = torch.ones(n, n, dtype=torch.bool).tril()
        if s["mask"] is not None:
            rows = [[w % (1 << 64) for w in row] for row in s["mask"][first : first + n].tolist()]
            drafts = torch.tensor([[row[i // 64] >> i % 64 & 1 for i in range(n)] for row in rows], dtype=torch.bool)
        hidden = torch.cat([torch.zeros(n, context, dtype=torch.bool), ~drafts], 1).cuda()
        for h in range(case["heads"]):
            k, v = (x[pages, h].reshape(-1, case["d"])[: context + n] for x in (keys, values))
            for g in range(h * group, (h + 1) * group):
                score = s["q"][first : first + n, g].double() @ k.t() / math.sqrt(case["d"])
                out[first : first + n, g] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v
    return out


def exact_adapter(case, s):
    out = s["x"].double() @ s["w"].double()
    if s["bias"] is not None:
        out += s["bias"].double()
    for i in range(case["adapters"]):
        rows = torch.nonzero(s["index"] == i).flatten()
        out[rows] += s["scale"][i].double() * (s["x"][rows].double() @ s["a"][i].double() @ s["b"][i].double())
    return out
