"""Run by test_state_edges_gpu.py in a process of its own: the first call that this process makes of
the library on the GPU is an eviction inside a capture."""
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "dist-gnn_amd",
                                "python"))
import torch  # noqa: E402

import dgs  # noqa: E402

gen = torch.Generator().manual_seed(0)
cols, budget = 300, 100
store0 = torch.randn(cols, 1, 1, 8, generator=gen).cuda()
w = torch.rand(1, 1, cols, generator=gen).cuda()
table = torch.randperm(cols, generator=gen).view(1, cols).cuda()
lens = torch.tensor([cols]).cuda()
store = store0.clone()


def step():
    return dgs.ops.evict_rows([store], w, None, table, lens, budget)


torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
for turn in range(3):
    w.copy_(torch.rand(1, 1, cols, generator=gen))
    store.copy_(store0)
    graph.replay()
    torch.cuda.synchronize()
    seen = [t.clone() for t in got] + [store.clone()]
    store.copy_(store0)
    want = list(step()) + [store]
    assert all(torch.equal(a, b) for a, b in zip(seen, want)), turn
dgs.ops._check_async_errors()
print("capture worker ok", flush=True)
