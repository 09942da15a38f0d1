"""Calls on rows captured in graphs: also a process's first call of the library, which makes the library's context."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# A process of its own, whose first call of the library is captured; then the same call without a graph.
FIRST = """
import sys
from types import SimpleNamespace
import torch
from orca_b200.packed import PackedRows
from orca_b200.lookup import lookup_grad, lookup_rows
dev = torch.device("cuda:0")
torch.manual_seed(0)
words = torch.randint(0, 1 << 12, (50, 24), device=dev).int()
words[:, :2] = 0x3d803e00            # (step 1/8, offset 1/16)
ids = lambda *s: torch.randint(1, 50, s, device=dev).int()
qt, edges, w = torch.randn(3, 1056, device=dev), torch.randn(50, 172, device=dev), torch.rand(172, device=dev)
table = (qt, ids(3, 200), ids(3, 200), torch.rand(3, 200, device=dev), edges, w)
a = SimpleNamespace(n_nodes=2, indptr=torch.tensor([0, 0, 400], device=dev), adj_nbr=ids(400), adj_eid=ids(400),
                    adj_ts=torch.arange(400, dtype=torch.float64, device=dev))
nodes, times = torch.ones(3, dtype=torch.int32, device=dev), torch.full((3,), 300.0, dtype=torch.float64, device=dev)
at, g = ids(5000), torch.randn(5000, 172, device=dev)
rows = PackedRows.from_words(words)
call = {"pull": lambda: rows.pull(at), "attend": lambda: rows.attend(*table),
        "attend_lists": lambda: rows.attend_lists(qt, a, nodes, times, edges, w), "lookup_rows": lambda: lookup_rows(edges, at, 0.5),
        "lookup_grad": lambda: lookup_grad(g, at, 50)}[sys.argv[1]]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = call()
graph.replay()
want = call()
torch.cuda.synchronize()
out, want = (x if isinstance(x, tuple) else (x,) for x in (out, want))
assert want[0].abs().sum() > 0 and all(torch.equal(x, y) for x, y in zip(out, want))
rows.check_status()
"""


@pytest.mark.parametrize("call", ["pull", "attend", "attend_lists", "lookup_rows", "lookup_grad"])
def test_a_process_first_call_is_captured(call):
    env = dict(os.environ, PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, "-c", FIRST, call], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_embeddings_over_packed_rows_captured():
    """Of a model whose weights are prepared: other nodes and times at every replay."""
    from helpers import graph
    from orca_b200.packed import PackedHistory
    from test_gpu_model import make_model
    dev = torch.device("cuda:0")
    g = graph("t_nb2")
    tgn = make_model(g)
    rs = np.random.RandomState(3)
    h = PackedHistory(g.n_nodes, 172, dev)
    h.push(torch.from_numpy(rs.randn(g.n_nodes, 172).astype(np.float32)).to(dev), np.arange(g.n_nodes))
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    at = [rs.randint(0, g.n_edges, 40) for _ in range(3)]
    inputs = [(up(g.sources[i].astype(np.int32)), up(g.timestamps[i])) for i in at]
    want = [tgn.packed_embeddings(h, *x, 10) for x in inputs]
    nodes, times = (x.clone() for x in inputs[0])
    graph_ = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph_):
        out = tgn.packed_embeddings(h, nodes, times, 10)
    for (n, t), y in list(zip(inputs, want))[::-1]:
        nodes.copy_(n), times.copy_(t)
        graph_.replay()
        assert torch.equal(out, y)
    h.check_status()
