"""Recorded calls whose scales change between replays, from ordinary ones to ones that take another part of the kernels and back: each
replay against the eager call, and against 64 bits."""

from __future__ import annotations

import pytest
import torch

from kernelcode_generate_amd import native
from tests.serving_util import adapter_oracle, assert_rows, f64, tree_oracle
from tests.test_gpu_adapter_matmul import Call as AdapterCall
from tests.test_gpu_tree_attention import Call as TreeCall

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


def recorded(calls):
    calls()  # (the workspace of the eager calls)
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    try:
        with torch.cuda.graph(graph, stream=stream):
            native.set_launch_mode(False, stream.cuda_stream)
            calls()
    finally:
        native.set_launch_mode(True, None)
    return graph


@pytest.mark.parametrize("m,k,n,count,rank", [(33, 2048, 320, 3, 64), (520, 512, 640, 3, 16), (600, 2048, 256, 3, 8), (4096, 544, 2048, 3, 16)])
def test_adapters_whose_range_changes(device, m, k, n, count, rank):
    call = AdapterCall(m, k, n, count, rank, F16)
    call.b = (call.b.float() * 2.0**-4).half()
    args = call.args(device)
    out = torch.empty(m, n, dtype=F16, device=device)
    graph = recorded(lambda: native.adapter_matmul(out, *args))
    plain = call.scale.clone()
    for powers in ((0, 0, 0), (14, 0, -18), (-18, -18, 14), (0, 0, 0), (14, 14, 14)):
        call.scale = plain * torch.exp2(torch.tensor(powers).float())
        args[6].copy_(call.scale)
        out.fill_(9.0)
        native.adapter_matmul(out, *args)
        eager = out.clone()
        out.fill_(0.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), powers
        expected, allowed = adapter_oracle(call.x, call.w, None, call.a, call.b, call.index, call.scale)
        small = torch.from_numpy((abs(expected) + allowed).max(1) < 65504)
        assert small.any()
        assert_rows(out.cpu()[small], expected[small.numpy()], allowed[small.numpy()], f"{powers}")


@pytest.mark.parametrize("cache", [E4M3, torch.int8])
@pytest.mark.parametrize("context,counts,group,d", [([900, 20], [1, 1], 4, 128), ([700, 3], [40, 9], 2, 64)])
def test_value_scales_that_change(device, cache, context, counts, group, d):
    call = TreeCall(context, counts, 2, group, d, 16, BF16, cache)
    args = call.args(device)
    out = call.out.to(device)
    graph = recorded(lambda: native.tree_attention(out, *args, call.scale))
    plain = call.vs.clone()
    signs = torch.randint(-1, 2, plain.shape, generator=torch.Generator().manual_seed(1)).float()
    for factor in (torch.ones_like(plain), signs, torch.full_like(plain, 2.0**-110), signs * 2.0**90, torch.ones_like(plain)):
        call.vs = plain * factor
        args[4].copy_(call.vs)
        out.fill_(9.0)
        native.tree_attention(out, *args, call.scale)
        eager = out.clone()
        out.fill_(0.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        power = float(factor.abs().max())  # (a power of two: the result is linear in the values)
        expected, allowed = tree_oracle(call.q, call.k, call.v, call.ks, call.vs / power, call.table, call.context.tolist(),
                                        call.starts.tolist(), call.mask, call.scale, call.out)
        allowed += 2.0**-134 / power  # half a subnormal step of the output
        assert_rows(torch.from_numpy(f64(out)) / power, expected, allowed)
