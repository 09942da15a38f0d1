"""Calls of a training step captured in graphs: also a process's first call of the library, and a whole step."""
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
import torch
from orca_b200.norm import layer_norm, layer_norm_grad
from orca_b200.optim import AdamW
dev = torch.device("cuda:0")
torch.manual_seed(0)
x, g, w, b = torch.randn(700, 172, device=dev), torch.randn(700, 172, device=dev), torch.rand(172, device=dev), torch.rand(172, device=dev)
wide = torch.randn(40, 20000, device=dev)
sets = [[torch.nn.Parameter(x.clone()), torch.nn.Parameter(w.clone())] for _ in range(2)]
opts = [AdamW(s, bits=8, max_norm=1.0) for s in sets]
for s in sets:
    s[0].grad, s[1].grad = g.clone(), b.clone()
def step(k):
    opts[k].step()
    return (*sets[k], *opts[k].moments()[0], *opts[k].moments()[1], opts[k].grad_norm)
call = {"layer_norm": lambda k: (layer_norm(x, w, b),), "layer_norm_grad": lambda k: layer_norm_grad(g, x, w), "wide": lambda k: layer_norm_grad(wide, wide),
        "adamw": step}[sys.argv[1]]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = call(0)
graph.replay()
want = call(1)
torch.cuda.synchronize()
assert want[0].abs().sum() > 0 and all(torch.equal(p, q) for p, q in zip(out, want))
"""


@pytest.mark.parametrize("call", ["layer_norm", "layer_norm_grad", "wide", "adamw"])
def test_a_process_first_call_is_captured(call):
    env = dict(os.environ, PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, "-c", FIRST, call], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_a_whole_step_captured():
    """Lookup, layer norm, gradients and AdamW in one graph, replayed with other ids: the same bits as one call after the other.  Two graphs of two
    optimisers, replayed in turn on two streams."""
    from orca_b200.lookup import lookup_grad, lookup_rows
    from orca_b200.norm import layer_norm, layer_norm_grad
    from orca_b200.optim import AdamW
    dev = torch.device("cuda:0")
    rs = np.random.RandomState(1)
    up = lambda *s: torch.from_numpy(rs.randn(*s).astype(np.float32)).to(dev)
    ids = [torch.from_numpy(rs.randint(0, 900, 3000)).to(dev) for _ in range(4)]
    start = up(900, 172), 1 + 0.1 * up(172), 0.1 * up(172)

    def make(bits):
        params = [torch.nn.Parameter(t.clone()) for t in start]
        for p in params:
            p.grad = torch.zeros_like(p)
        return params, AdamW(params, 1e-2, max_norm=1.0, bits=bits)

    def step(params, opt, at):
        with torch.no_grad():
            table, w, b = params
            x = lookup_rows(table, at, 0.5, padding=0)
            y = layer_norm(x, w, b)
            dx, dw, db = layer_norm_grad(y, x, w)
            table.grad.copy_(lookup_grad(dx, at, 900, 0.5, padding=0))
            w.grad.copy_(dw)
            b.grad.copy_(db)
            opt.step()

    want, graphs = [], []
    for bits in (32, 8):
        params, opt = make(bits)
        for at in ids:
            step(params, opt, at)
        want.append(params)
        params, opt = make(bits)
        held, graph = ids[0].clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(params, opt, held)
        graphs.append((params, opt, held, graph, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for at in ids:
        for _, _, held, graph, stream in graphs:
            with torch.cuda.stream(stream):
                held.copy_(at)
                graph.replay()
    torch.cuda.synchronize()
    for (params, opt, *_), w in zip(graphs, want):
        assert int(opt.state[params[0]]["step"]) == 4
        assert all(torch.equal(p, q) for p, q in zip(params, w))
