"""Block tables that stay on the device between steps (8-bit KV cache).

With ``kv_dtype="fp8"`` a step does not upload its requests' block tables.  Each sequence owns a
row of one resident table; the runner sends the lengths, the row numbers and the blocks that the
step adds, and :func:`lightbulb_b200.ops.step_tables` enters them and builds the step's tables,
slots, positions and attention work list.  A host mirror tells which rows no longer hold what the
block manager says (a new sequence, copy-on-write, blocks freed and taken again): those rows are
uploaded before the step.
"""
from __future__ import annotations

from collections import OrderedDict
from typing import List, Tuple

import numpy as np
import torch


class ResidentTables:
    def __init__(self, rows: int, width: int, device):
        self.tables = torch.zeros(rows, width, dtype=torch.int32, device=device)
        self.mirror = np.zeros((rows, width), dtype=np.int32)
        self.row_of: "OrderedDict[int, int]" = OrderedDict()   # least recently used first
        self.free = list(range(rows - 1, -1, -1))
        self.uploads = 0                                       # rows uploaded so far

    def grow(self, rows: int) -> None:
        """Room for ``rows`` sequences in a step.  The device table moves: what was captured with
        the old one has to be captured again."""
        more = rows - len(self.mirror)
        if more <= 0:
            return
        width = self.mirror.shape[1]
        self.free += list(range(rows - 1, len(self.mirror) - 1, -1))
        self.mirror = np.concatenate([self.mirror, np.zeros((more, width), np.int32)])
        self.tables = torch.cat([self.tables, self.tables.new_zeros(more, width)])

    def _rows(self, seq_ids: List[int]) -> np.ndarray:
        batch = set(seq_ids)
        out = np.empty(len(seq_ids), dtype=np.int64)
        for i, sid in enumerate(seq_ids):
            row = self.row_of.pop(sid, None)
            if row is None:
                if not self.free:
                    old = next((s for s in self.row_of if s not in batch), None)
                    if old is None:
                        raise ValueError(f"{len(seq_ids)} sequences in a step, "
                                         f"{len(self.mirror)} resident rows")
                    self.free.append(self.row_of.pop(old))
                row = self.free.pop()
            self.row_of[sid] = row
            out[i] = row
        return out

    def place(self, seq_ids: List[int], host: np.ndarray, ctx: np.ndarray, q: np.ndarray,
              block_size: int) -> Tuple[np.ndarray, np.ndarray]:
        """``host`` [B, W]: the block manager's tables after this step's blocks were added;
        ``ctx`` / ``q``: cached and new tokens.  Returns the requests' rows and the step's new
        blocks in request order."""
        rows = self._rows(seq_ids)
        w = host.shape[1]
        col = np.arange(w)
        have = -(-ctx // block_size)
        need = -(-(ctx + q) // block_size)
        old = col < have[:, None]
        stale = ((self.mirror[rows, :w] != host) & old).any(1)
        if stale.any():
            r = rows[stale]
            self.mirror[r, :w] = np.where(old[stale], host[stale], self.mirror[r, :w])
            idx = torch.from_numpy(r).to(self.tables.device)
            self.tables[idx] = torch.from_numpy(self.mirror[r]).to(self.tables.device)
            self.uploads += len(r)
        new = ~old & (col < need[:, None])
        part = self.mirror[rows, :w]
        part[new] = host[new]                 # what the device enters this step
        self.mirror[rows, :w] = part
        return rows.astype(np.int32), host[new]
