"""Page tables of the request slots on the device, and a step's maps made from them (csrc/page_tables.cu)."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import native
from ..cache.slots import SLOT_WORDS
from ..errors import KernelError
from .native import c_int, c_void_p, pointer

native.register_library(
    "b200_page_tables", ("page_tables.cu",),
    {
        "b200_page_table_set": [c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p, c_int, c_void_p],
        "b200_step_maps": [c_void_p, c_int, c_int] + [c_void_p] * 4 + [c_int] + [c_void_p] * 4 + [c_int, c_int, c_int, c_void_p],
        "b200_slot_load_maps": [c_void_p, c_int] + [c_void_p] * 5 + [c_int, c_int, c_void_p] + [c_int] * 3 + [c_void_p],
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

    here = native.current_device()
    at = pointer(tables, "tables", here, torch.int32, dims=2)
    rows_at = pointer(rows, "rows", here, torch.int32, dims=1)
    shape = rows.shape
    columns_at, pages_at = pointer(columns, "columns", here, torch.int32, shape=shape), pointer(pages, "pages", here, torch.int32, shape=shape)
    slots, width = tables.shape
    if not slots or not width:
        raise KernelError(f"a page table of shape {tuple(tables.shape)} has no cells")
    if shape[0]:
        native.call("b200_page_table_set", at, slots, width, rows_at, columns_at, pages_at, shape[0], native.stream_ptr())


def step_maps(
    tables: torch.Tensor, *, slots: torch.Tensor, kv_len: torch.Tensor, counts: torch.Tensor, page_size: int, num_tokens: int,
    width: int | None = None, out: StepMaps | None = None,
) -> StepMaps:
    """The maps of a step whose entry ``r`` is the request in row ``slots[r]`` of ``tables``, with ``counts[r]`` new tokens and
    ``kv_len[r]`` tokens once the step has run (int32, on the device); ``num_tokens``: the sum of the counts.  The block table is
    ``width`` columns wide (``None``: as wide as ``tables``); cells behind an entry's last page are -1, whatever ``tables`` holds
    there.  An entry of length 0 (a row that pads the batch) has an empty row; its tokens have positions from 0 on and no slot.

    ``out``: tensors to write into, which may have room for more entries and tokens than there are (those are left as they are);
    what is ``None`` there is not made."""

    here = native.current_device()
    at = pointer(tables, "tables", here, torch.int32, dims=2)
    slots_at = pointer(slots, "slots", here, torch.int32, dims=1)
    entries = slots.shape[0]
    kv_len_at, counts_at = pointer(kv_len, "kv_len", here, torch.int32, shape=(entries,)), pointer(counts, "counts", here, torch.int32, shape=(entries,))
    table_rows, table_width = tables.shape
    if (not table_rows or not table_width or not 0 < page_size < 1 << 31 or not 0 <= num_tokens < 1 << 31
            or (width is not None and not 0 < width < 1 << 31)):
        raise KernelError(f"tables {tuple(tables.shape)}, page_size {page_size}, num_tokens {num_tokens} and width {width} do not fit")
    if out is None:
        # the three short ones in one piece of memory
        q_start, positions, token_entry = tables.new_empty(entries + 1 + 2 * num_tokens).split_with_sizes(
            (entries + 1, num_tokens, num_tokens))
        out = StepMaps(tables.new_empty((entries, width or table_width)), q_start, positions, token_entry,
                       tables.new_empty(num_tokens, dtype=torch.int64))
        pointers = [t.data_ptr() for t in (out.block_table, q_start, positions, token_entry, out.slot_map)]
    else:
        if width is not None and isinstance(out.block_table, torch.Tensor) and out.block_table.shape[-1] != width:
            raise KernelError(f"out.block_table has {out.block_table.shape[-1]} columns, not {width}")
        pointers = []
        for name, dtype, dims, least in (("block_table", torch.int32, 2, entries), ("q_start", torch.int32, 1, entries + 1),
                                         ("positions", torch.int32, 1, num_tokens), ("token_entry", torch.int32, 1, num_tokens),
                                         ("slot_map", torch.int64, 1, num_tokens)):
            t = getattr(out, name)
            if t is None and dims == 1:
                pointers.append(None)
                continue
            pointers.append(pointer(t, f"out.{name}", here, dtype, dims=dims, align=dtype.itemsize))
            if t.shape[0] < least:
                raise KernelError(f"out.{name} has room for {t.shape[0]}, {least} are needed")
    if not entries:
        if out.q_start is not None:
            out.q_start[:1].zero_()       # the sum over no entries
    else:
        native.call("b200_step_maps", at, table_rows, table_width, slots_at, kv_len_at, counts_at, pointers[0], out.block_table.shape[1],
                    *pointers[1:], entries, int(page_size), int(num_tokens), native.stream_ptr())
    return out


def slot_load_maps(records: torch.Tensor, slots: torch.Tensor, token_ids: torch.Tensor, positions: torch.Tensor, kv_len: torch.Tensor, *,
                   tables: torch.Tensor, page_size: int, block_table: torch.Tensor) -> None:
    """``slots.slot_load`` (a decode batch's token ids, positions and lengths from the records of its slots, whose positions
    advance) and the batch's ``block_table`` from ``tables`` by those lengths, as ``step_maps`` makes it, in one launch.  The slots
    of live records are distinct."""

    here = native.current_device()
    at = pointer(records, "records", here, torch.int32, dims=2)
    if records.shape[1] != SLOT_WORDS:
        raise KernelError(f"records of {records.shape[1]} words are not slot records")
    n = slots.shape[0]
    given = [pointer(t, name, here, torch.int32, shape=(n,)) for t, name in ((slots, "slots"), (token_ids, "token_ids"), (positions, "positions"),
                                                                     (kv_len, "kv_len"))]
    tables_at, block_at = pointer(tables, "tables", here, torch.int32, dims=2), pointer(block_table, "block_table", here, torch.int32, dims=2)
    if tables.numel() == 0 or block_table.shape[0] < n or block_table.shape[1] == 0 or not 0 < page_size < 1 << 31:
        raise KernelError(f"tables {tuple(tables.shape)}, block_table {tuple(block_table.shape)} and page_size {page_size} do not fit {n} slots")
    native.call("b200_slot_load_maps", at, records.shape[0], *given, tables_at, tables.shape[0], tables.shape[1], block_at,
                block_table.shape[1], n, int(page_size), native.stream_ptr())
