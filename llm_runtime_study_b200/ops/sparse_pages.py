"""Attention over the pages of the cache that a query chooses by a cheap score (csrc/sparse_pages.cu, csrc/sparse_attention.cu), one build
per head size.

``page_bounds`` keeps, beside the pages of keys, the least and the greatest value of every channel on each full page;
``choose_pages`` ranks the pages a query row sees by an upper bound of its scores on them; ``paged_attention_chosen`` attends
to the keys of the pages chosen.  What a row chooses, and what it gets, depends on its position and the cache alone, not on
the batch or on where a prompt was cut.
"""

from __future__ import annotations

import torch

from . import native
from ..errors import KernelError
from .native import c_float, c_int, c_void_p, ptr, require, require_here, stream_ptr, tag

_TABLE = {
    "b200_sparse_pages_head_dim": [],
    "b200_page_bounds": [c_void_p] * 3 + [c_int] + [c_void_p] * 2 + [c_int] * 6 + [c_void_p],
    "b200_choose_pages": [c_void_p] * 5 + [c_int, c_void_p] + [c_int] * 12 + [c_void_p],
    "b200_attend_chosen": [c_void_p] * 7 + [c_int, c_void_p] + [c_int] * 7 + [c_float, c_int, c_int, c_void_p],
}
SOURCES = ("sparse_pages.cu", "sparse_attention.cu")
DTYPES = (torch.float32, torch.bfloat16)
MAX_TABLE_WIDTH = 51200      # pages of a row whose scores fit into a CTA's shared memory


def supported(head_dim: int) -> bool:
    return head_dim % 16 == 0 and 16 <= head_dim <= 256


def library_name(head_dim: int) -> str:
    if not supported(head_dim):
        raise KernelError(f"head size {head_dim} is not a multiple of 16 up to 256")
    name = f"b200_sparse_pages_d{head_dim}"
    if name not in native.library_specs():
        native.register_library(name, SOURCES, _TABLE, defines=(f"HEAD_DIM={head_dim}",))
    return name


def build(head_dim: int) -> None:
    """Compile the kernels for one head size."""

    from ..csrc.build import build_library

    name = library_name(head_dim)
    build_library(name, SOURCES, native.library_defines(name))


def _pool(t: torch.Tensor, name: str, dims: int, dtype=None) -> tuple[int, ...]:
    require(t, name, dtype=dtype or DTYPES, dims=dims)
    require_here(t, name, 16)
    if t.numel() == 0:
        raise KernelError(f"{name} of shape {tuple(t.shape)} holds nothing")
    return tuple(t.shape)


def _rows(positions, token_entry, block_table, n: int) -> None:
    require(positions, "positions", dtype=torch.int32, shape=(n,))
    require(token_entry, "token_entry", dtype=torch.int32, shape=(n,))
    require(block_table, "block_table", dtype=torch.int32, dims=2)
    if block_table.numel() == 0:
        raise KernelError(f"a block table of shape {tuple(block_table.shape)} has no cells")
    for t, name in ((positions, "positions"), (token_entry, "token_entry"), (block_table, "block_table")):
        require_here(t, name)


def _query(q: torch.Tensor, kv_heads: int, head_dim: int, dtype) -> tuple[int, int]:
    require(q, "q", dtype=dtype, dims=3)
    require_here(q, "q", 16)
    n, heads, d = q.shape
    if d != head_dim or heads == 0 or heads % kv_heads:
        raise KernelError(f"q {tuple(q.shape)} does not fit {kv_heads} key heads of {head_dim}")
    if n * heads >= 1 << 31:
        raise KernelError(f"{n} rows of {heads} heads are too many for one launch")
    return n, heads


def page_bounds(keys: torch.Tensor, bounds: torch.Tensor, *, block_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
                max_q_len: int) -> None:
    """Write the bounds of every page that became full in this step: entry ``e`` (a row of ``block_table``) holds ``kv_len[e]``
    tokens now, the last ``q_start[e + 1] - q_start[e]`` of them new.  ``keys`` ``[pages, kv heads, page size, d]``, ``bounds``
    ``[pages, kv heads, 2, d]`` (low, high) of the same type; ``max_q_len``: the most new tokens of an entry (a hint for the
    launch).  Pages that are not full keep what they have; a NaN among a channel's keys makes both bounds NaN."""

    pages, kv_heads, page_size, d = _pool(keys, "keys", 4)
    library = library_name(d)
    require(bounds, "bounds", dtype=keys.dtype, shape=(pages, kv_heads, 2, d))
    require_here(bounds, "bounds", 16)
    require(kv_len, "kv_len", dtype=torch.int32, dims=1)
    entries = kv_len.shape[0]
    require(block_table, "block_table", dtype=torch.int32, dims=2)
    require(q_start, "q_start", dtype=torch.int32, shape=(entries + 1,))
    for t, name in ((block_table, "block_table"), (q_start, "q_start"), (kv_len, "kv_len")):
        require_here(t, name)
    if block_table.shape[0] != entries or block_table.numel() == 0 and entries:
        raise KernelError(f"a block table of shape {tuple(block_table.shape)} does not fit {entries} entries")
    if max_q_len < 0:
        raise KernelError("max_q_len must not be negative")
    if not entries or not max_q_len:
        return
    native.call("b200_page_bounds", ptr(keys), ptr(bounds), ptr(block_table), block_table.shape[1], ptr(q_start), ptr(kv_len), entries,
                -(-max_q_len // page_size), kv_heads, page_size, pages, tag(keys.dtype), stream_ptr(), library=library)


def choose_shape(rows: int, entries: int, kv_heads: int, width: int, head_dim: int) -> tuple[int, int]:
    """(tiles of eight rows or not, CTAs of a cluster) of a choice.  Tiles where entries have several rows each; a cluster shares out
    the pages of few rows, and the shared memory that the scores of many pages need."""

    def fill(units: int, cluster: int) -> int:
        while cluster < 8 and 2 * cluster * units <= 2 * native.sm_count() and width // (2 * cluster) >= 64:
            cluster *= 2
        return cluster

    if rows >= 2 * entries:
        sums, cluster = 2 * head_dim * 64, 1
        while cluster < 8 and sums + 32 * width // cluster > 100 * 1024:
            cluster *= 2
        if sums + 32 * width // cluster <= 200 * 1024:
            return 1, fill(-(-rows // 8) * kv_heads, cluster)
    return 0, fill(rows * kv_heads, 1)


def choose_pages(q: torch.Tensor, bounds: torch.Tensor, *, positions: torch.Tensor, token_entry: torch.Tensor, block_table: torch.Tensor,
                 page_size: int, budget: int, first: int = 1, last: int = 1) -> torch.Tensor:
    """For every row of ``q`` ``[n, heads, d]`` and every kv head, which of the pages ``0 .. positions[i] // page_size`` of entry
    ``token_entry[i]`` it should read: int32 ``[n, kv heads, budget]``, columns of the block table in rising order, -1 behind
    them.  The ``first`` pages and the ``last`` ones (at least one: the row's own, whose bounds are not up to date) are always
    among them; the others have the highest ``sum over the group's heads and channels of max(q low, q high)``, formed as
    ``sum_c high_c sum_h max(q_hc, 0) + low_c sum_h min(q_hc, 0)`` in 64 bits and rounded to 32; of equal scores the lower page is
    taken, a NaN (an infinite bound that meets a sum of 0 gives one) ranks first.  A page that is not held (an id that is none) is
    not chosen."""

    pages, kv_heads, two, d = _pool(bounds, "bounds", 4)
    library = library_name(d)
    if two != 2:
        raise KernelError(f"bounds of shape {tuple(bounds.shape)} are not [pages, kv heads, 2, d]")
    n, heads = _query(q, kv_heads, d, bounds.dtype)
    _rows(positions, token_entry, block_table, n)
    if page_size <= 0 or first < 0 or last < 1 or budget < first + last:
        raise KernelError(f"page_size {page_size}, budget {budget}, first {first} and last {last}: the budget holds the first pages and "
                          "the last ones, of which there is one at least")
    if block_table.shape[1] > MAX_TABLE_WIDTH:
        raise KernelError(f"block tables of more than {MAX_TABLE_WIDTH} pages are not taken: {block_table.shape[1]}")
    if n * kv_heads * budget >= 1 << 40:
        raise KernelError(f"a budget of {budget} pages for {n} rows of {kv_heads} heads is too much")
    chosen = torch.empty((n, kv_heads, budget), dtype=torch.int32, device=q.device)
    if n:
        native.call("b200_choose_pages", ptr(q), ptr(bounds), ptr(positions), ptr(token_entry), ptr(block_table), block_table.shape[1],
                    ptr(chosen), n, block_table.shape[0], heads, kv_heads, int(page_size), pages, int(budget), int(first), int(last),
                    *choose_shape(n, block_table.shape[0], kv_heads, block_table.shape[1], d), tag(q.dtype), stream_ptr(), library=library)
    return chosen


def attention_parts(rows: int, heads: int, kv_heads: int, budget: int, page_size: int, dtype: torch.dtype) -> int:
    """Into how many CTAs of a cluster the list of a row and kv head is cut: 1, 2, 4 or 8.  float32: from the list's length alone, so
    that the order of the sums does not depend on the batch.  bfloat16: until the GPU is full, no part shorter than 128 keys."""

    keys, parts = budget * page_size, 1
    if dtype == torch.float32:
        while parts < 8 and 2 * parts <= budget and keys // (2 * parts) >= 256:
            parts *= 2
        return parts
    ctas = rows * kv_heads * -(-(heads // kv_heads) // 8)
    while parts < 8 and 2 * parts <= budget and keys // (2 * parts) >= 128 and 2 * parts * ctas <= 2 * native.sm_count():
        parts *= 2
    return parts


def paged_attention_chosen(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, chosen: torch.Tensor, *, positions: torch.Tensor,
                           token_entry: torch.Tensor, block_table: torch.Tensor, scale: float) -> torch.Tensor:
    """Attention of row ``i`` of ``q`` ``[n, heads, d]`` over the keys of the pages ``chosen[i, kv head]`` (columns of row
    ``token_entry[i]`` of the block table, distinct, in any order; -1: none) at positions up to ``positions[i]``.  ``keys`` and
    ``values`` are ``[pages, kv heads, page size, d]``.  Keys behind the position and pages that are not held are neither read nor
    counted; a row without a key (or without a score above minus infinity) gives zeros."""

    pages, kv_heads, page_size, d = _pool(keys, "keys", 4)
    library = library_name(d)
    require(values, "values", dtype=keys.dtype, shape=keys.shape)
    require_here(values, "values", 16)
    n, heads = _query(q, kv_heads, d, keys.dtype)
    _rows(positions, token_entry, block_table, n)
    require(chosen, "chosen", dtype=torch.int32, dims=3)
    require_here(chosen, "chosen")
    if tuple(chosen.shape[:2]) != (n, kv_heads) or chosen.shape[2] == 0:
        raise KernelError(f"chosen of shape {tuple(chosen.shape)} does not fit {n} rows of {kv_heads} key heads")
    if chosen.shape[2] * page_size > 1 << 30:
        raise KernelError(f"{chosen.shape[2]} pages of {page_size} tokens a row are too many")
    out = torch.empty_like(q)
    if n:
        native.call("b200_attend_chosen", ptr(q), ptr(keys), ptr(values), ptr(chosen), ptr(positions), ptr(token_entry), ptr(block_table),
                    block_table.shape[1], ptr(out), n, block_table.shape[0], heads, kv_heads, page_size, pages, chosen.shape[2],
                    float(scale), attention_parts(n, heads, kv_heads, chosen.shape[2], page_size, q.dtype), tag(q.dtype), stream_ptr(),
                    library=library)
    return out
