"""Page tables of the request slots on the device, and a step's maps made from them (csrc/page_tables.cu)."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import native
from ..errors import KernelError
from .native import c_int, c_void_p, ptr, require

native.register_library(
    "b200_page_tables", ("page_tables.cu",),
    {
        "b200_page_table_set": [c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p, c_int, c_void_p],
        "b200_step_maps": [c_void_p, c_int, c_int] + [c_void_p] * 4 + [c_int] + [c_void_p] * 4 + [c_int, c_int, c_int, c_void_p],
    },
)


@dataclass
class StepMaps:
    """What a step needs to know of its tokens, on the device.  ``None``: not wanted."""

    block_table: torch.Tensor                   # [entries, width] int32: the pages of every entry, -1 behind its last one
    q_start: torch.Tensor | None = None         # [entries + 1] int32: first token of every entry
    positions: torch.Tensor | None = None       # [tokens] int32
    token_entry: torch.Tensor | None = None     # [tokens] int32
    slot_map: torch.Tensor | None = None        # [tokens] int64: row of the pool's ``[pages * page_size]`` rows, -1 without a page


def page_table_set(tables: torch.Tensor, *, rows: torch.Tensor, columns: torch.Tensor, pages: torch.Tensor) -> None:
    """``tables[rows[i], columns[i]] = pages[i]`` (all int32, the cells distinct); a cell outside the table is left out."""

    native.require_here(tables, "tables")
    require(tables, "tables", dtype=torch.int32, dims=2)
    require(rows, "rows", dtype=torch.int32, dims=1)
    for t, name in ((columns, "columns"), (pages, "pages")):
        require(t, name, dtype=torch.int32, shape=rows.shape)
    for t, name in ((rows, "rows"), (columns, "columns"), (pages, "pages")):
        native.require_here(t, name)
    if tables.numel() == 0:
        raise KernelError(f"a page table of shape {tuple(tables.shape)} has no cells")
    if rows.shape[0] == 0:
        return
    native.call("b200_page_table_set", ptr(tables), tables.shape[0], tables.shape[1], ptr(rows), ptr(columns), ptr(pages),
                rows.shape[0], native.stream_ptr())


def step_maps(
    tables: torch.Tensor, *, slots: torch.Tensor, kv_len: torch.Tensor, counts: torch.Tensor, page_size: int, num_tokens: int,
    width: int | None = None, out: StepMaps | None = None,
) -> StepMaps:
    """The maps of a step whose entry ``r`` is the request in row ``slots[r]`` of ``tables``, with ``counts[r]`` new tokens and
    ``kv_len[r]`` tokens once the step has run (int32, on the device); ``num_tokens``: the sum of the counts.  The block table is
    ``width`` columns wide (``None``: as wide as ``tables``); cells behind an entry's last page are -1, whatever ``tables`` holds
    there.  An entry of length 0 (a row that pads the batch) has an empty row, its tokens position 0 and no slot.

    ``out``: tensors to write into, which may have room for more entries and tokens than there are (those are left as they are);
    what is ``None`` there is not made."""

    native.require_here(tables, "tables")
    require(tables, "tables", dtype=torch.int32, dims=2)
    require(slots, "slots", dtype=torch.int32, dims=1)
    entries = slots.shape[0]
    for t, name in ((kv_len, "kv_len"), (counts, "counts")):
        require(t, name, dtype=torch.int32, shape=(entries,))
    if tables.numel() == 0 or page_size <= 0 or num_tokens < 0 or (width is not None and width <= 0):
        raise KernelError(f"tables {tuple(tables.shape)}, page_size {page_size}, num_tokens {num_tokens} and width {width} do not fit")
    if out is None:
        def ints(*shape, dtype=torch.int32):
            return torch.empty(shape, dtype=dtype, device=tables.device)

        out = StepMaps(ints(entries, tables.shape[1] if width is None else width), ints(entries + 1), ints(num_tokens),
                       ints(num_tokens), ints(num_tokens, dtype=torch.int64))
        if entries == 0:
            out.q_start.zero_()
    elif width is not None and out.block_table.shape[-1] != width:
        raise KernelError(f"out.block_table has {out.block_table.shape[-1]} columns, not {width}")
    require(out.block_table, "out.block_table", dtype=torch.int32, dims=2)
    for t, name, least, dtype in ((out.block_table, "block_table", entries, torch.int32), (out.q_start, "q_start", entries + 1, torch.int32),
                                  (out.positions, "positions", num_tokens, torch.int32),
                                  (out.token_entry, "token_entry", num_tokens, torch.int32),
                                  (out.slot_map, "slot_map", num_tokens, torch.int64)):
        if t is None:
            continue
        require(t, f"out.{name}", dtype=dtype, dims=2 if t is out.block_table else 1)
        if t.shape[0] < least:
            raise KernelError(f"out.{name} has room for {t.shape[0]}, {least} are needed")
    for t, name in ((slots, "slots"), (kv_len, "kv_len"), (counts, "counts"), (out.block_table, "out.block_table")):
        native.require_here(t, name)
    if entries == 0:
        return out
    native.call("b200_step_maps", ptr(tables), tables.shape[0], tables.shape[1], ptr(slots), ptr(kv_len), ptr(counts),
                ptr(out.block_table), out.block_table.shape[1], ptr(out.q_start), ptr(out.positions), ptr(out.token_entry),
                ptr(out.slot_map), entries, int(page_size), int(num_tokens), native.stream_ptr())
    return out
