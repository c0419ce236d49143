"""The block tables of all request slots on the device, kept in step with the host's.

The reference rebuilds a batch's block table on the host for every step (mini_llm/cache/paged/cache.py:179-183).  Here each
group of pages has a table ``[slots + 1, width]`` on the device; a step sends the cells that changed since the last one (pages
taken, pages that a window has given back) and its rows are put together there (``ops/page_tables.py``), so what goes to the
device does not grow with the length of the sequences.  Cells behind a request's last page hold whatever an earlier request
left: the rows of a step are cut by its lengths.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence

import numpy as np
import torch


@dataclass
class _Known:
    """What the device's row of a slot holds of the request that has it."""

    request: int
    columns: list[int]      # per group: leading columns that are there
    given_back: list[int]   # per group: leading columns known to hold no page any more


class DeviceTables:
    def __init__(self, slots: int, widths: Sequence[int], device: torch.device) -> None:
        # the last row belongs to nobody: the rows that pad a batch point there
        self.tensors = [torch.full((slots + 1, width), -1, dtype=torch.int32, device=device) for width in widths]
        self._known: dict[int, _Known] = {}

    def current(self, requests: Sequence) -> bool:
        """Whether the device's rows of these requests are the host's already (what most decode steps find)."""

        for request in requests:
            known = self._known.get(request.slot)
            if known is None or known.request != request.id:
                return False
            for table, columns, back in zip(request.tables, known.columns, known.given_back):
                if columns != len(table) or (back < columns and table[back] < 0):
                    return False
        return True

    def changes(self, requests: Sequence) -> list[np.ndarray]:
        """The cells that differ from what the device holds: for every group their rows, columns and pages (int32)."""

        groups = len(self.tensors)
        rows: list[list[int]] = [[] for _ in range(groups)]
        columns: list[list[int]] = [[] for _ in range(groups)]
        pages: list[list[int]] = [[] for _ in range(groups)]
        for request in requests:
            known = self._known.get(request.slot)
            if known is None or known.request != request.id:
                known = _Known(request.id, [0] * groups, [0] * groups)
            for g, table in enumerate(request.tables):
                at, back = known.columns[g], known.given_back[g]
                if at > len(table):
                    at = back = 0
                if at < len(table):
                    columns[g].extend(range(at, len(table)))
                    pages[g].extend(table[at:])
                while back < at and table[back] < 0:
                    columns[g].append(back)
                    pages[g].append(-1)
                    back += 1
                rows[g].extend([request.slot] * (len(columns[g]) - len(rows[g])))
        return [np.asarray(cells[g], dtype=np.int32) for g in range(groups) for cells in (rows, columns, pages)]

    def sent(self, requests: Sequence) -> None:
        """The changes of these requests are on their way to the device, before everything that is launched from now on."""

        for request in requests:
            known = self._known.get(request.slot)
            if known is None or known.request != request.id:
                known = self._known[request.slot] = _Known(request.id, [0] * len(self.tensors), [0] * len(self.tensors))
            for g, table in enumerate(request.tables):
                known.columns[g] = len(table)
                back = min(known.given_back[g], len(table))
                while back < len(table) and table[back] < 0:
                    back += 1
                known.given_back[g] = back
