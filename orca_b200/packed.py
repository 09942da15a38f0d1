"""Rows of 172 values held in 4 bits: a table of 96 bytes a row instead of 688, put into, read from and attended over by node id.

``PackedRows`` is such a table (edge features, node features, embeddings); ``PackedHistory`` is the historical-embedding cache of
modules/history.py:4-46 in this form: in the same memory it keeps 6.7 times the nodes (105 bytes a node with what push and the flags
need, against 701).  The reference has no counterpart, its cache is fp32.  A value is off by at most half a step of its group, a step
being a fifteenth of the range that the group's 128 or 44 values span (include/orca_b200.h has the format).
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib
from .history import History


def _host_ids(inds, limit, what):
    """A host list of ids as int32, refused where one lies outside the table."""
    ids = np.asarray(inds)
    if ids.size and ids.dtype.kind not in "iu":
        raise TypeError(f"{what} must be integers, got {ids.dtype}")
    if ids.size and (int(ids.min()) < 0 or int(ids.max()) >= limit):
        raise _lib.OrcaError(_lib.E_BOUNDS, f"{what}: ids from {int(ids.min())} to {int(ids.max())} for a table of {limit} rows")
    return torch.from_numpy(np.ascontiguousarray(ids, dtype=np.int32))


def _fp32(edges):
    if not isinstance(edges, torch.Tensor) or edges.dtype is not torch.float32:
        raise ValueError("edges are PackedRows, or a contiguous fp32 tensor [edges, 172]")
    return edges


class PackedRows:
    """``num_rows`` rows of 172 values in 4 bits on a CUDA device, all zero at first.

    ``words`` is the table, int32 ``[num_rows, 24]``.  Ids on the device are not looked at by the calls: rows outside the table
    are left out (zeros for ``pull``) and reported, which ``check_status`` raises; ids from the host are checked by the call.
    All calls enqueue on the current stream and return.  A table may be read by any number of streams at a time; ``push`` changes it
    and is ordered by the caller.  Calls may be captured in a graph, but a table's first ``push``.

    Nothing here has a gradient: rows that are pushed are taken as they are, attention refuses an input that asks for one."""

    def __init__(self, num_rows, device="cuda"):
        num_rows = int(num_rows)
        if not 0 < num_rows < 1 << 31:
            raise ValueError(f"a table has 1 to 2^31 - 1 rows, not {num_rows}")
        self._adopt(torch.zeros(num_rows, _lib.PACKED_WORDS, dtype=torch.int32, device=_lib.require_cuda(device)))

    def _adopt(self, words):
        self.words, self.device, self.num_rows = words, words.device, words.shape[0]
        self.status = torch.zeros(4, dtype=torch.int32, device=words.device)
        self._record = None       # last positions of pushed ids (all zero between calls), made by the first push

    @classmethod
    def from_words(cls, words):
        """The table over words that are there (int32 [rows, 24], contiguous); they are not copied."""
        if not (isinstance(words, torch.Tensor) and words.is_cuda and words.dtype == torch.int32 and words.dim() == 2
                and words.shape[1] == _lib.PACKED_WORDS and words.is_contiguous() and words.shape[0] > 0
                and words.data_ptr() % 16 == 0):
            raise ValueError("packed rows are a contiguous CUDA tensor, int32 [rows, 24], 16-byte aligned")
        self = cls.__new__(cls)
        self._adopt(words)
        return self

    @classmethod
    def of(cls, table):
        """The rows of a whole table ([n, 172] in fp32, bf16 or fp16) in 4 bits."""
        table = cls._rows(table, table.device)
        self = cls(table.shape[0], table.device)
        self._fill(table)
        return self

    def _fill(self, table):
        _lib.rows().push(self.words, self.status, None, table, None)

    @staticmethod
    def _rows(x, device):
        if not isinstance(x, torch.Tensor) or x.dim() != 2 or x.shape[1] != _lib.DIM:
            raise ValueError("rows are a tensor [n, 172]")
        if x.device != device or x.dtype not in _lib.TYPES:
            x = x.detach().to(device, x.dtype if x.dtype in _lib.TYPES else torch.float32)
        return x if x.stride(1) == 1 and x.stride(0) >= _lib.DIM else x.detach().contiguous()

    def _ids(self, inds):
        if not isinstance(inds, torch.Tensor) or not inds.is_cuda:
            return _host_ids(inds, self.num_rows, "ids").reshape(-1).to(self.device)
        if inds.dtype != torch.int32:
            if inds.dtype != torch.int64:
                raise TypeError(f"ids must be int32 or int64, got {inds.dtype}")
            inds = inds.clamp(-1, 0x7fffffff)      # (what does not fit must not come back as another id)
        if inds.device != self.device or inds.dtype != torch.int32:
            inds = inds.to(self.device, torch.int32)
        return inds if inds.dim() == 1 and inds.is_contiguous() else inds.reshape(-1).contiguous()

    def reset_parameters(self):
        self.words.zero_()

    def push(self, x, inds):
        """Puts x[i] at row inds[i] (modules/history.py:38-40); among equal ids the last one's row stays."""
        ids, x = self._ids(inds), self._rows(x, self.device)
        if self._record is None:
            with torch.cuda.device(self.device):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the first push into a table makes what later ones need: call one before capturing a graph")
                self._record = torch.zeros(self.num_rows, dtype=torch.int32, device=self.device)
        _lib.rows().push(self.words, self.status, self._record, x, ids)

    def pull(self, inds):
        """The rows `inds` in fp32, [m, 172] (modules/history.py:32-36)."""
        return _lib.rows().pull(self.words, self.status, self._ids(inds))

    def push_and_pull(self, x, push_inds, pull_inds):
        """modules/history.py:42-46."""
        self.push(x, push_inds)
        return self.pull(pull_inds)

    def attend(self, qt, nbr, eid, delta, edges, time_w):
        """Attention of a layer (model/temporal_attention.py:43-53) over neighbours whose rows are this table's.

        qt     [n, 1056] fp32, the projected queries (orca_attn_query)
        nbr, eid, delta  [n, k] int32, int32, fp32: neighbour (0: no slot), edge and time difference of each slot, any k
        edges  features by edge id: PackedRows, or [edges, 172] fp32
        time_w [172] fp32, the weights of the time encoding
        Returns ctx [n, 1032] fp32, the weighted sums of [neighbour | edge | time] per head, and valid [n] uint8; a row without
        slots is zero and not valid.  A value is decoded with an error of half a step of fp32 of sixteen steps of its group and then rounded
        (pull only rounds); magnitudes times 2^12 times a row's slots have to stay within fp32."""
        return _lib.rows().attend(self.words, self.status, qt, edges.words if isinstance(edges, PackedRows) else _fp32(edges), time_w,
                                  nbr, eid, delta)

    def attend_lists(self, qt, finder, nodes, timestamps, edges, time_w, last=None):
        """The same over whole histories: the slots of query i are the interactions of nodes[i] strictly before timestamps[i]
        in the adjacency of `finder` (a NeighborFinder, or an object with its n_nodes, indptr, adj_nbr, adj_eid and adj_ts: contiguous,
        with indptr within the others), the `last` of them (None: all)."""
        if last is not None and int(last) < 1:
            raise ValueError(f"last is a number of interactions from 1, or None for all, not {last}")
        d = self.device
        ids, ts = nodes, timestamps
        if not isinstance(ids, torch.Tensor) or not ids.is_cuda:
            ids = _host_ids(ids, finder.n_nodes, "nodes").to(d)
        elif ids.dtype is not torch.int32:
            if ids.dtype is not torch.int64:
                raise TypeError(f"nodes must be int32 or int64, got {ids.dtype}")
            ids = ids.clamp(-1, 0x7fffffff).to(d, torch.int32)
        if not isinstance(ts, torch.Tensor):
            ts = torch.from_numpy(np.array(ts, dtype=np.float64))
        if ts.dtype is not torch.float64 or ts.device != d or ids.device != d:
            ids, ts = ids.to(d), ts.to(d, torch.float64)
        if ids.dim() != 1 or ts.dim() != 1:
            ids, ts = ids.reshape(-1), ts.reshape(-1)
        return _lib.rows().attend_lists(self.words, self.status, qt, edges.words if isinstance(edges, PackedRows) else _fp32(edges), time_w,
                                        finder.indptr, finder.adj_nbr, finder.adj_eid, finder.adj_ts, finder.n_nodes, ids, ts,
                                        0 if last is None else int(last))

    def check_status(self):
        """Waits for the current stream and raises if a kernel met an id outside a table since the last check."""
        code, _, _, detail = self.status.tolist()
        if code:
            self.status.zero_()
            raise _lib.OrcaError(code, f"an id outside its table was left out (query or position {detail})")


class PackedHistory(History):
    """The historical-embedding cache with its rows in 4 bits (``rows``, a PackedRows) behind the interface of ``History``.  The
    model's own batches keep fp32 histories and refuse this one; ``TGN.packed_embeddings`` reads it."""

    def _make_table(self):
        # (PackedRows.push keeps the last of equal ids by itself)
        self.rows = PackedRows(self.num_embeddings, self._device)

    @property
    def emb(self):
        """All rows in fp32, a copy; assigning packs."""
        return self.rows.pull(torch.arange(self.num_embeddings, dtype=torch.int32, device=self._device))

    @emb.setter
    def emb(self, table):
        if tuple(table.shape) != (self.num_embeddings, self.embedding_dim):
            raise ValueError(f"the table is [{self.num_embeddings}, {self.embedding_dim}]")
        self.rows._fill(self.rows._rows(table, self._device))

    def reset_parameters(self):
        self.rows.reset_parameters()

    def detach_history(self):
        pass

    def pull(self, inds):
        return self.rows.pull(inds)

    def push(self, x, inds):
        self.rows.push(x, inds)

    def push_and_pull(self, x, push_inds, pull_inds):
        return self.rows.push_and_pull(x, push_inds, pull_inds)

    def attend(self, qt, nbr, eid, delta, edges, time_w):
        return self.rows.attend(qt, nbr, eid, delta, edges, time_w)

    def attend_lists(self, qt, finder, nodes, timestamps, edges, time_w, last=None):
        return self.rows.attend_lists(qt, finder, nodes, timestamps, edges, time_w, last)

    def check_status(self):
        self.rows.check_status()
