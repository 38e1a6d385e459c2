"""Calls recorded where recordings hold all the workspace that they may have, down to the last bytes: which form was recorded is told by the
number of the graph's nodes."""

from __future__ import annotations

import ctypes
import gc
import random

import pytest
import torch

from kernelcode_generate_amd import native
from tests.step_util import assert_close, assign_oracle, int8_oracle

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32
PAGE, ROWS = 16, 5000


def runtime():
    """The HIP runtime that is loaded already."""

    with open("/proc/self/maps") as maps:
        return ctypes.CDLL(next(line.split()[-1] for line in maps if "libamdhip64" in line))


class Recorder:
    def __init__(self):
        self.hip, self.stream, self.graphs = runtime(), torch.cuda.Stream(), []
        self.hip.hipGraphGetNodes.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_size_t)]
        self.stream.wait_stream(torch.cuda.current_stream())

    def __call__(self, call):
        """(graph, its number of nodes), kept until the recorder goes."""

        graph = torch.cuda.CUDAGraph(keep_graph=True)
        try:
            with torch.cuda.graph(graph, stream=self.stream):
                native.set_launch_mode(False, self.stream.cuda_stream)
                call()
        finally:
            native.set_launch_mode(True, None)
        count = ctypes.c_size_t()
        assert self.hip.hipGraphGetNodes(graph.raw_cuda_graph(), None, ctypes.byref(count)) == 0
        self.graphs.append(graph)
        return graph, count.value


class Pages:
    """Requests whose tokens are more rows than one launch assigns where there is a workspace."""

    def __init__(self, device, requests, seed=0):
        rng = random.Random(seed)
        self.requests, self.start = requests, [rng.randrange(0, 40) for _ in range(requests)]
        self.added = [rng.randrange(0, 2 * ROWS // requests + 2) for _ in range(requests)]
        per = max(-(-(c + n) // PAGE) for c, n in zip(self.start, self.added))
        pages = list(range(requests * per))
        rng.shuffle(pages)
        held = [-(-c // PAGE) for c in self.start]
        self.old = [[pages.pop() if p < h else -1 for p in range(per)] for h in held]
        self.stack = pages
        self.slots, self.positions, self.starts = (torch.zeros(n, dtype=t, device=device) for n, t in ((ROWS, torch.int64), (ROWS, I32), (requests + 1, I32)))
        self.table, self.free, self.count, self.context, self.new = (torch.tensor(x, dtype=I32, device=device) for x in (
            self.old, self.stack, [len(self.stack)], self.start, self.added))

    def run(self):
        native.kv_cache_assign(self.slots, self.positions, self.starts, self.table, self.free, self.count, self.context, self.new, PAGE)

    def check(self, replay):
        self.table.copy_(torch.tensor(self.old, dtype=I32))
        self.count.fill_(len(self.stack))
        for t in (self.slots, self.positions, self.starts):
            t.fill_(-5)
        replay()
        torch.cuda.synchronize()
        want = assign_oracle(self.old, self.stack, len(self.stack), self.start, self.added, PAGE, ROWS)
        assert [t.tolist() for t in (self.slots, self.positions, self.starts, self.table)] == list(want[:4]) and self.count.item() == want[4]


def test_pages_and_long_sums_without_a_workspace(device):
    record = Recorder()
    big, w = torch.zeros(16000, 4096, dtype=BF16, device=device), torch.ones(16, 4096, dtype=torch.int8, device=device)
    out, one = torch.empty(16000, 16, dtype=BF16, device=device), torch.ones(16, device=device)
    pages = {requests: Pages(device, requests) for requests in (8192, 1000, 100, 20, 3)}
    gc.collect()
    torch.cuda.synchronize()
    pages[3].run()  # an eager call that takes a workspace frees those of graphs that are gone
    recorded = {requests: [record(p.run)] for requests, p in pages.items()}
    assert all(r[0][1] == 2 for r in recorded.values())  # with a workspace: the sums, then the rows
    for m in (16000, 4000, 1000, 250, 60, 10, 2):  # 65 MB and less a recording; then a call of each size of pages until it gets none
        for _ in range(17 if m == 16000 else 5):
            record(lambda: native.int8_matmul(out[:m], big[:m], None, w, one))
    for requests, p in pages.items():
        for _ in range(200):
            recorded[requests].append(record(p.run))
            if recorded[requests][-1][1] == 1:
                break
        assert recorded[requests][-1][1] == 1, f"{requests} requests: a workspace is left"
    # products in one launch: 131071 products of 2^14 a sum, of codes whose rows are no whole pieces
    values = torch.full((3, 131071), -128, dtype=torch.int8)
    weight, scales = torch.full((70, 131071), -128, dtype=torch.int8), (torch.full((3,), 0.01), torch.full((70,), 0.001))
    x, wide, xs, ws, got = values.to(device), weight.to(device), *(s.to(device) for s in scales), torch.zeros(3, 70, device=device)
    product, nodes = record(lambda: native.int8_matmul(got, x, xs, wide, ws))
    assert nodes == 1
    want = int8_oracle(values.long().numpy(), scales[0].numpy(), weight, scales[1], None, torch.float32)
    for turn in range(3):
        for requests, p in pages.items():
            p.check(recorded[requests][-1][0].replay)  # one launch
            p.check(recorded[requests][0][0].replay)  # two
            p.check(p.run)  # eager, on the stream's own workspace
        got.zero_()
        product.replay()
        torch.cuda.synchronize()
        assert_close(got, *want, f"turn {turn}")
