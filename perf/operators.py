"""Rows of node tables by their ids: held in 4 bits, attended over, and looked up for training.

What a user of temporal graph models does beside scoring a stream of edges:

``attend``        The attention of a layer over historical embeddings held in 4 bits: every query row names its slots in a table of
                  neighbours (``PackedRows.attend``), as the layers of the model do.
``attend_lists``  The same over all interactions that a node had before a time, straight from the time-sorted adjacency
                  (``PackedRows.attend_lists``): lists from none to hundreds of thousands of slots.
``push_pull``     Rows are put into the 4-bit table and rows are read from it (``PackedRows.push_and_pull``).
``lookup``        Rows of a trained table by id, times a scale, and the gradient of the table (``lookup_rows``).

A row of 172 values in 4 bits is 24 words of 32 bits.  Word 0 says how columns 0..127 are held, word 1 the same of columns
128..171: the step (bfloat16) in the low half, the offset (bfloat16) in the high half.  The codes follow, eight columns a word, the
first in the lowest bits.  A value is offset + step * code.  The offset is the largest bfloat16 that no value of the group
is below, the step the smallest bfloat16 that is at least (largest - offset) / 15, a code the nearest integer (ties to even) to (value -
offset) / step.  A group with a NaN, or a value of 2^126 or more, is NaN.

Sizes are those of the synthetic workloads in ``orca_b200/synthetic.py`` (batches of 200 to 2000 edges, 10 or 20 neighbours, up to
1,140,149 nodes) and ranges around them.  Neighbour 0 is the padding of a table.
"""
import math
import types

import numpy as np
import torch

own = False

D = 172                 # columns of a row
GROUP = 128             # columns of a row's first group
WORDS = 24              # words of a packed row
KEY = 3 * D             # [neighbour | edge | time]
HEAD = 528              # floats from one head's query to the next
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2, "packed": 96}


# ---------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one node is asked for, as it arrives at a service
        dict(name="attend_one", op="attend", rows=1, k=10, nodes=9227, edges=157474, edge="packed", empty=0.0),
        # the endpoints of a batch of 2000 edges with their negatives; edge features as the model holds them
        dict(name="attend_batch", op="attend", rows=6000, k=10, nodes=194086, edges=1443340, edge="float32", empty=0.2),
        # a group of batches on the largest graph, twenty neighbours, everything in 4 bits
        dict(name="attend_group", op="attend", rows=66001, k=20, nodes=1140150, edges=2000001, edge="packed", empty=0.1),
        # the whole histories of a small batch's endpoints
        dict(name="lists_small", op="attend_lists", lists=37, mean=33, spread=1.0, nodes=9228, edges=157475, edge="packed"),
        # three hubs of a large graph
        dict(name="lists_hubs", op="attend_lists", lists=3, mean=400000, spread=0.5, nodes=1140150, edges=1200001, edge="packed"),
        # whole histories of many nodes; lengths over three orders of magnitude
        dict(name="lists_large", op="attend_lists", lists=4001, mean=480, spread=1.3, nodes=1140150, edges=2000001, edge="packed"),
        # the same with edge features in 32 bits
        dict(name="lists_edges32", op="attend_lists", lists=1201, mean=250, spread=1.0, nodes=194086, edges=1443340, edge="float32"),
        # the rows of one batch of 200 edges go to the history and come back with their neighbours
        dict(name="push_batch", op="push_pull", rows=600, pulled=2600, nodes=9228, type="float32"),
        # a table is filled and read in bulk, from rows in 16 bits
        dict(name="push_bulk", op="push_pull", rows=399999, pulled=500001, nodes=1140150, type="bfloat16"),
        # a training step's rows of one small batch
        dict(name="lookup_batch", op="lookup", ids=600, nodes=9228, width=172, type="float32", skew=1.5, scale=1.0, grad=True),
        # features in 16 bits of a large batch's neighbours: hubs come up thousands of times
        dict(name="lookup_hubs", op="lookup", ids=60001, nodes=194086, width=172, type="bfloat16", skew=3.0, scale=0.5, grad=True),
        # a training step on the largest graph
        dict(name="lookup_large", op="lookup", ids=399999, nodes=1140150, width=172, type="float32", skew=1.5, scale=13.114877, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend_lists", "attend_lists", "push_pull", "lookup", "lookup"])
    nodes = _log(rng, 1500, 1140150)
    if op == "attend":
        k = rng.choice([1, 5, 10, 10, 20, 20, 32, rng.randint(2, 200)])
        return dict(op=op, rows=_log(rng, 1, min(66001, 1300000 // k)), k=k, nodes=nodes, edges=_log(rng, 20000, 2000001),
                    edge=rng.choice(["packed", "float32"]), empty=round(rng.uniform(0.0, 0.6), 2))
    if op == "attend_lists":
        edge = rng.choice(["packed", "packed", "float32"])
        lists = _log(rng, 1, 4001)
        return dict(op=op, lists=lists, mean=_log(rng, 2, min(400000, (1900000 if edge == "packed" else 300000) // lists)),
                    spread=round(rng.uniform(0.2, 1.3), 2), nodes=nodes, edges=_log(rng, 20000, 2000001), edge=edge)
    if op == "push_pull":
        return dict(op=op, rows=_log(rng, 1, 399999), pulled=_log(rng, 1, 500001), nodes=nodes, type=rng.choice(list(TYPES)))
    return dict(op=op, ids=_log(rng, 1, 399999), nodes=nodes, width=rng.choice([172, 172, rng.randint(1, 172)]),
                type=rng.choice(list(TYPES)), skew=round(rng.uniform(1.0, 4.0), 2), scale=round(rng.uniform(0.1, 14.0), 3),
                grad=rng.random() < 0.75)


def _distinct(picks, of):
    """Expected number of different ones among so many picks."""
    return of * -math.expm1(-picks / of)


def work(case):
    op = case["op"]
    if op in ("attend", "attend_lists"):
        if op == "attend":
            rows, slots = case["rows"], case["rows"] * case["k"] * (1 - case["empty"])
            index = case["rows"] * case["k"] * 12        # neighbour, edge, time difference
        else:
            rows, slots = case["lists"], case["lists"] * case["mean"] * (1 - WITHIN / 2)
            index = slots * 16 + rows * 28               # neighbour, edge, time; node, time, where its list is
        data = _distinct(slots, case["nodes"]) * 96 + _distinct(slots, case["edges"]) * (96 if case["edge"] == "packed" else 4 * D)
        # two heads: a product and a weighted sum over the columns of a slot
        return {"bytes": rows * 2 * (2 * KEY * 4) + index + data, "flops": slots * 2 * KEY * 4}
    if op == "push_pull":
        size = SIZE[case["type"]]
        return {"bytes": case["rows"] * (4 + D * size) + _distinct(case["rows"], case["nodes"]) * 96
                + case["pulled"] * (4 + 4 * D) + _distinct(case["pulled"], case["nodes"]) * 96,
                "flops": (case["rows"] + case["pulled"]) * D * 2}
    row = case["width"] * SIZE[case["type"]]
    read = sum(_distinct(case["ids"] / 16, case["nodes"] * (((i + 1) / 16) ** case["skew"] - (i / 16) ** case["skew"])) for i in range(16))
    b = case["ids"] * (4 + row) + read * row
    f = case["ids"] * case["width"]
    if case["grad"]:
        b += case["ids"] * row + case["nodes"] * row
        f *= 2
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------------------------------------- inputs
WITHIN = 0.25      # the share of queries that lie within their node's times; the others come after all of them


def _time_weights():
    return torch.from_numpy((1 / 10 ** np.linspace(0, 9, D)).astype(np.float32)).cuda()


def _ids(n, nodes, gen, skew=1.0, low=1):
    """Ids from low up to nodes - 1; the larger skew, the more often the small ones."""
    u = torch.rand(n, dtype=torch.float64, device="cuda", generator=gen)
    return (low + (u ** skew * (nodes - low)).long()).clamp_(max=nodes - 1)


def _random_words(n, gen):
    """A table as it is after training: rows of unit size with their own offsets; row 0 is zero."""
    words = torch.randint(-2 ** 31, 2 ** 31, (n, WORDS), dtype=torch.int64, device="cuda", generator=gen)
    words[:, -1] &= 0xffff                     # (the last word holds four columns)
    for g in range(2):
        step = (0.2 + 0.3 * torch.rand(n, device="cuda", generator=gen)).bfloat16()
        offset = (-7.5 * step.float() + 0.2 * torch.randn(n, device="cuda", generator=gen)).bfloat16()
        words[:, g] = (step.view(torch.int16).long() & 0xffff) | (offset.view(torch.int16).long() << 16)
    words[0] = 0
    return words.to(torch.int32)


def _edge_rows(case, gen):
    if case["edge"] == "packed":
        return _random_words(case["edges"], gen)
    t = torch.randn(case["edges"], D, device="cuda", generator=gen)
    t[0] = 0
    return t


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    rand = lambda *s: torch.rand(*s, dtype=torch.float64, device="cuda", generator=gen)
    op, n = case["op"], case["nodes"]
    s = types.SimpleNamespace(op=op)
    if op in ("attend", "attend_lists"):
        s.words, s.edges, s.time_w = _random_words(n, gen), _edge_rows(case, gen), _time_weights()
        rows = case["rows"] if op == "attend" else case["lists"]
        s.qt = torch.zeros(rows, 2 * HEAD, device="cuda")
        for h in range(2):
            s.qt[:, h * HEAD:h * HEAD + KEY] = randn(rows, KEY) * (2 / math.sqrt(KEY))
        if op == "attend":
            k = case["k"]
            # tables are padded in front; some rows have no neighbour at all
            have = (k - (rand(rows) * (2 * case["empty"] * (k + 1))).long()).clamp_(min=0)
            have = torch.where(rand(rows) < 0.05 * (case["empty"] > 0), 0, have)
            used = torch.arange(k, device="cuda") >= k - have[:, None]
            s.nbr = torch.where(used, _ids(rows * k, n, gen, 1.5).view(rows, k), 0).int()
            s.eid = torch.where(used, _ids(rows * k, case["edges"], gen).view(rows, k), 0).int()
            s.delta = torch.where(used, torch.exp(rand(rows, k) * 19), 1e8).float()
        else:
            # interactions of the nodes that are asked for, each node's in the order of time
            s.nodes = _ids(rows, n, gen).int()
            length = torch.exp(case["spread"] * randn(rows).double() - case["spread"] ** 2 / 2)
            length = (length / length.mean() * case["mean"]).round().long().clamp_(min=1)
            per_node = torch.zeros(n, dtype=torch.long, device="cuda")
            per_node.scatter_reduce_(0, s.nodes.long(), length, "amax")      # (a node asked for twice has one list)
            indptr = torch.zeros(n + 1, dtype=torch.long, device="cuda")
            indptr[1:] = per_node.cumsum(0)
            total = int(indptr[-1])
            span = 2.0e8
            owner = torch.repeat_interleave(torch.arange(n, device="cuda"), per_node)
            ts = torch.sort(owner * (2 * span) + (rand(total) * span).floor())[0] - owner * (2 * span)
            s.adjacency = types.SimpleNamespace(n_nodes=n, indptr=indptr, adj_ts=ts, adj_nbr=_ids(total, n, gen, 1.5).int(),
                                                adj_eid=_ids(total, case["edges"], gen).int())
            # most ask now, behind all interactions; others at a time between them, or before the first
            s.times = torch.where(rand(rows) < WITHIN, rand(rows), 1 + rand(rows) / 10)
            s.times = (s.times * span).floor()
        if own:
            from orca_b200.packed import PackedRows
            s.rows = PackedRows.from_words(s.words)
            s.edge_rows = PackedRows.from_words(s.edges) if case["edge"] == "packed" else s.edges
    elif op == "push_pull":
        s.words = _random_words(n, gen)
        s.x = (randn(case["rows"], D) * torch.exp(0.5 * randn(case["rows"], 1)) + 0.3 * randn(1, D)).to(TYPES[case["type"]])
        s.ids = _ids(case["rows"], n, gen, 1.5).int()
        fresh = torch.cat([s.ids, _ids(case["pulled"], n, gen, low=0).int()])
        s.pulled = fresh[:case["pulled"]].contiguous()
        if own:
            from orca_b200.packed import PackedRows
            s.rows = PackedRows.from_words(s.words)
    else:
        t = TYPES[case["type"]]
        s.table = randn(n, case["width"]).to(t)
        s.table[0] = 0
        s.ids = _ids(case["ids"], n, gen, case["skew"], low=0).int()
        s.scale, s.grad = case["scale"], None
        if case["grad"]:
            s.grad = randn(case["ids"], case["width"]).to(t)
            s.table.requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------- the plain forms
def _decode(words):
    """The values of packed rows, in 32 bits: [..., 24] int32 -> [..., 172]."""
    codes = (words[..., 2:, None] >> (4 * torch.arange(8, device=words.device))) & 15
    codes = codes.flatten(-2)[..., :D].float()
    step, offset = ((words[..., :2] << 16).view(torch.float32), (words[..., :2] & -65536).view(torch.float32))
    first = torch.arange(D, device=words.device) < GROUP
    return torch.where(first, codes * step[..., :1] + offset[..., :1], codes * step[..., 1:] + offset[..., 1:])


def _round_bf16(bits, up):
    """32-bit floats given by their bits, moved to a bfloat16: away from zero where `up` and a bit is lost, else towards it."""
    return torch.where(up & ((bits & 0xffff) != 0), (bits & -65536) + 65536, bits & -65536)


def _encode(x):
    """Packed rows of [m, 172] values.  In 64 bits: a quotient next to a border between two codes belongs on one side of it."""
    words = torch.zeros(x.shape[0], WORDS, dtype=torch.int64, device=x.device)
    codes = []
    for g, v in enumerate((x[:, :GROUP], x[:, GROUP:])):
        v = v.double()
        fine = (v.abs() < 2.0 ** 126).all(1)
        v = torch.where(fine[:, None], v, 0.0)
        bits = v.amin(1).float().view(torch.int32)
        offset = _round_bf16(bits, bits < 0)
        low = offset.view(torch.float32).double()
        wide = (v.amax(1) - low) / 15
        near = wide.float()
        bits = near.view(torch.int32) + (near.double() < wide).int()
        step = _round_bf16(bits, bits >= 0)
        size = step.view(torch.float32).double()[:, None]
        codes.append(torch.where(size > 0, torch.round((v - low[:, None]) / torch.where(size > 0, size, 1.0)), 0.0).long())
        word = ((step >> 16) & 0xffff) | (offset & -65536)
        words[:, g] = torch.where(fine, word, 0x7fc07fc0)
    codes = torch.cat(codes + [torch.zeros(x.shape[0], 4, dtype=torch.int64, device=x.device)], 1).view(-1, 22, 8)
    words[:, 2:] = (codes << (4 * torch.arange(8, device=x.device))).sum(2)
    return words.to(torch.int32)          # (the low 32 bits)


def _keys(s, nbr, eid, delta):
    """[neighbour | edge | time] of slots.  The angle is the product in 32 bits, as the model's time encoder has it; its cosine is
    taken in 64 bits, since angles reach 2e8."""
    edge = _decode(s.edges[eid]) if s.edges.dtype == torch.int32 else s.edges[eid]
    return torch.cat([_decode(s.words[nbr]), edge, torch.cos((delta[..., None] * s.time_w).double()).float()], -1)


def _queries(s):
    return torch.stack([s.qt[:, :KEY], s.qt[:, HEAD:HEAD + KEY]], 1)       # [rows, 2, 516]


def _attend(s):
    x, q = _keys(s, s.nbr.long(), s.eid.long(), s.delta), _queries(s)
    used = (s.nbr != 0)[:, None, :]
    logits = torch.where(used, torch.matmul(q, x.transpose(1, 2)), -math.inf)
    top = logits.amax(2, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(2, keepdim=True)
    out = torch.matmul(p, x) / torch.where(total == 0, 1.0, total)
    return out.flatten(1), used.any(2).flatten().to(torch.uint8)


def _slots(s):
    """The slots of all lists, one behind the other: where they lie, and whose they are."""
    a, nodes = s.adjacency, s.nodes.long()
    before = torch.zeros(len(a.adj_ts) + 1, dtype=torch.long, device="cuda")
    beg, end = a.indptr[nodes], a.indptr[nodes + 1]
    # interactions before the time: each node's times rise, and 4e8 a node keeps the nodes apart
    owner = torch.repeat_interleave(torch.arange(a.n_nodes, device="cuda"), a.indptr[1:] - a.indptr[:-1])
    count = torch.searchsorted(owner * 4e8 + a.adj_ts, nodes * 4e8 + s.times) - beg
    count = torch.minimum(count.clamp(min=0), end - beg)
    row = torch.repeat_interleave(torch.arange(len(nodes), device="cuda"), count)
    first = count.cumsum(0) - count
    return beg[row] + torch.arange(len(row), device="cuda") - first[row], row, count


def _attend_lists(s):
    at, row, count = _slots(s)
    a, rows = s.adjacency, len(s.nodes)
    delta = (s.times[row] - a.adj_ts[at].float().double()).float()
    x, q = _keys(s, a.adj_nbr[at].long(), a.adj_eid[at].long(), delta), _queries(s)
    out = torch.zeros(rows, 2, KEY, dtype=torch.float64, device="cuda")
    for h in range(2):                                                     # (the heads: one at a time for room)
        logit = (x * q[row, h]).sum(1)
        top = torch.full((rows,), -math.inf, device="cuda").scatter_reduce_(0, row, logit, "amax")
        p = torch.exp(logit - top[row]).double()                           # (sums over up to a million slots: in 64 bits)
        total = torch.zeros(rows, dtype=torch.float64, device="cuda").index_add_(0, row, p)
        out[:, h].index_add_(0, row, x * p[:, None])
        out[:, h] /= torch.where(total == 0, 1.0, total)[:, None]
    return out.float().flatten(1), (count > 0).to(torch.uint8)


def _push_pull(s):
    ids, m = s.ids.long(), len(s.ids)
    at = torch.arange(m, device="cuda")
    last = torch.full((len(s.words),), -1, device="cuda").scatter_reduce_(0, ids, at, "amax")   # the last of equal ids stays
    wins = last[ids] == at
    s.words[ids[wins]] = _encode(s.x[wins])
    return _decode(s.words[s.pulled.long()])


def _lookup(s):
    ids = s.ids.long()
    out = (s.table.detach()[ids].float() * s.scale).to(s.table.dtype)
    if s.grad is None:
        return out
    # (sums over up to tens of thousands of rows: in 64 bits); row 0 is padding and learns nothing
    g = torch.zeros(s.table.shape, dtype=torch.float64, device="cuda").index_add_(0, ids, s.grad.double())
    g[0] = 0
    return out, (g * s.scale).to(s.table.dtype)


def run(state):
    s = state
    if not own:
        return {"attend": _attend, "attend_lists": _attend_lists, "push_pull": _push_pull, "lookup": _lookup}[s.op](s)
    if s.op == "attend":
        return s.rows.attend(s.qt, s.nbr, s.eid, s.delta, s.edge_rows, s.time_w)
    if s.op == "attend_lists":
        return s.rows.attend_lists(s.qt, s.adjacency, s.nodes, s.times, s.edge_rows, s.time_w)
    if s.op == "push_pull":
        return s.rows.push_and_pull(s.x, s.ids, s.pulled)
    from orca_b200.lookup import lookup_rows
    out = lookup_rows(s.table, s.ids, scale=s.scale, padding=0)
    return out if s.grad is None else (out.detach(), torch.autograd.grad(out, s.table, s.grad)[0])


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits
def _value64(words):
    """[m, 24] int32 -> [m, 172] float64, a column at a time from its word, shift and group."""
    col = torch.arange(D, device=words.device)
    code = torch.bitwise_and(torch.bitwise_right_shift(words[:, 2 + col // 8].long(), 4 * (col % 8)), 15).double()
    how = words[:, (col >= GROUP).long()].contiguous()
    parts = how.view(torch.bfloat16).view(len(words), D, 2).double()       # (the low half comes first)
    return parts[..., 1] + parts[..., 0] * code


def _edge64(s, eid):
    return _value64(s.edges[eid]) if s.edges.dtype == torch.int32 else s.edges[eid].double()


def _exact_rows(s, lo, hi):
    """Rows lo..hi of a table of neighbours, the weights of padding set to nothing behind the softmax of what is left."""
    nbr, eid, delta = s.nbr[lo:hi].long(), s.eid[lo:hi].long(), s.delta[lo:hi]
    x = torch.cat([_value64(s.words[nbr.flatten()]), _edge64(s, eid.flatten()),
                   torch.cos(torch.outer(delta.flatten(), s.time_w).double())], 1).view(*nbr.shape, KEY)
    q = s.qt[lo:hi].double()
    logits = torch.einsum("rhc,rkc->rhk", torch.stack([q[:, :KEY], q[:, HEAD:HEAD + KEY]], 1), x)
    some = (nbr != 0).any(1)
    logits[(some[:, None] & (nbr == 0))[:, None].expand_as(logits)] = -math.inf
    w = torch.softmax(logits, -1) * some[:, None, None]
    return torch.einsum("rhk,rkc->rhc", w, x).flatten(1), some.to(torch.uint8)


def _exact_list(s, r, beg, end, time):
    """One list: its interactions before the time, by themselves."""
    a = s.adjacency
    n = int((a.adj_ts[beg:end] < time).sum())
    if n == 0:
        return torch.zeros(2 * KEY, dtype=torch.float64, device="cuda"), 0
    delta = (time - a.adj_ts[beg:beg + n].float().double()).float()
    x = torch.cat([_value64(s.words[a.adj_nbr[beg:beg + n].long()]), _edge64(s, a.adj_eid[beg:beg + n].long()),
                   torch.cos(torch.outer(delta, s.time_w).double())], 1)
    q = s.qt[r].double()
    return (torch.softmax(torch.stack([q[:KEY], q[HEAD:HEAD + KEY]]) @ x.T, -1) @ x).flatten(), 1


def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "attend":
        step = max(1, 100000 // case["k"])
        parts = [_exact_rows(s, i, i + step) for i in range(0, case["rows"], step)]
        return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
    if s.op == "attend_lists":
        nodes, times, ptr = s.nodes.tolist(), s.times.tolist(), s.adjacency.indptr.tolist()
        parts = [_exact_list(s, r, ptr[v], ptr[v + 1], t) for r, (v, t) in enumerate(zip(nodes, times))]
        return torch.stack([p[0] for p in parts]), torch.tensor([p[1] for p in parts], dtype=torch.uint8, device="cuda")
    if s.op == "push_pull":
        # the row that each pulled id was given last, in the steps that its group has
        ids, x = s.ids.long().cpu().numpy(), s.x.double()
        order = np.argsort(ids, kind="stable")
        ends = np.flatnonzero(np.append(ids[order][1:] != ids[order][:-1], True))
        holder = np.full(case["nodes"], -1, dtype=np.int64)
        holder[ids[order][ends]] = order[ends]
        of = torch.from_numpy(holder).cuda()[s.pulled.long()]
        held = _value64(s.words[s.pulled.long()])
        v = x[of.clamp(min=0)]
        for c in (slice(0, GROUP), slice(GROUP, D)):
            g = v[:, c]
            low = g.min(1, keepdim=True).values
            near = low.bfloat16()                      # (nearest; one bfloat16 further down where that lies above)
            down = torch.nextafter(near, torch.full_like(near, -math.inf))
            low = torch.where(near.double() > low, down, near).double()
            step = (g.max(1, keepdim=True).values - low) / 15
            near = step.bfloat16()
            step = torch.where(near.double() < step, torch.nextafter(near, torch.full_like(near, math.inf)), near).double()
            v[:, c] = torch.where(step > 0, low + step * ((g - low) / step).round(), low)
        return torch.where((of >= 0)[:, None], v, held)
    ids = s.ids.long()
    out = s.table.detach().double()[ids] * s.scale
    if s.grad is None:
        return out
    # rows of equal ids side by side, each stretch summed
    order = torch.argsort(ids, stable=True)
    lengths = torch.bincount(ids, minlength=case["nodes"])
    g = torch.segment_reduce(s.grad.double()[order], "sum", lengths=lengths, axis=0, initial=0) * s.scale
    g[0] = 0
    return out, g
