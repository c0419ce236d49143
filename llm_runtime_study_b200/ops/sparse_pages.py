"""Attention over the pages of the cache that a query chooses by a cheap score (csrc/sparse_pages.cu, csrc/sparse_attention.cu), one build
per head size.

``page_bounds`` keeps, beside the pages of keys, the least and the greatest value of every channel on each full page;
``choose_pages`` ranks the pages a query row sees by an upper bound of its scores on them; ``paged_attention_chosen`` attends
to the keys of the pages chosen.

What a row chooses depends on its query, its position and the cache, not on the batch or on where a prompt was cut, as far as
64-bit sums go: rows of prompts and single tokens have their scores added up in different orders, so a score that lies within the
rounding of those sums of a midpoint between two 32-bit numbers may come out one step apart.  What float32 attention makes of a choice
does not depend on the batch; in bfloat16 the number of rows decides how a list is cut and so the order of its sums (within the
rounding of the output).
"""

from __future__ import annotations

from functools import lru_cache

import torch

from . import native
from ..errors import KernelError
from .native import c_float, c_int, c_void_p, pointer, stream_ptr

_TABLE = {
    "b200_sparse_pages_head_dim": [],
    "b200_page_bounds": [c_void_p] * 3 + [c_int] + [c_void_p] * 2 + [c_int] * 6 + [c_void_p],
    "b200_choose_pages": [c_void_p] * 5 + [c_int, c_void_p] + [c_int] * 11 + [c_void_p],
    "b200_choose_pages_tiles": [c_void_p] * 5 + [c_int, c_void_p] + [c_int] * 11 + [c_void_p],
    "b200_attend_chosen": [c_void_p] * 7 + [c_int, c_void_p] + [c_int] * 7 + [c_float, c_int, c_int, c_int, c_void_p],
}
SOURCES = ("sparse_pages.cu", "sparse_attention.cu")
DTYPES = (torch.float32, torch.bfloat16)
MAX_SIZE = 1 << 30           # of a page or a list
MAX_TABLE_WIDTH = 51200      # pages of a row whose scores fit into a CTA's shared memory


def supported(head_dim: int) -> bool:
    return head_dim % 16 == 0 and 16 <= head_dim <= 256


@lru_cache(maxsize=None)
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


def _pool(t: torch.Tensor, name: str, here: int) -> int:
    """The address of pages of keys, which set the type of everything beside them."""

    if not isinstance(t, torch.Tensor) or t.dtype not in native.DTYPE_TAG:
        native.require(t, name, dtype=DTYPES)
    return pointer(t, name, here, t.dtype, dims=4, align=16)


def _sizes(*sizes: int) -> None:
    if min(sizes) <= 0:
        raise KernelError(f"pages of sizes {sizes} hold nothing")


def _rows(positions, token_entry, block_table, n: int, here: int) -> tuple[int, int, int, int]:
    """Addresses of the rows' positions and entries and of the block table, and the table's width."""

    given = (pointer(positions, "positions", here, torch.int32, shape=(n,)), pointer(token_entry, "token_entry", here, torch.int32, shape=(n,)),
             pointer(block_table, "block_table", here, torch.int32, dims=2), block_table.shape[1])
    if not block_table.numel():
        raise KernelError(f"a block table of shape {tuple(block_table.shape)} has no cells")
    return given


def _query(q: torch.Tensor, kv_heads: int, head_dim: int, dtype, here: int) -> tuple[int, int, int]:
    at = pointer(q, "q", here, dtype, dims=3, align=16)
    n, heads, d = q.shape
    if d != head_dim or heads == 0 or heads % kv_heads:
        raise KernelError(f"q {tuple(q.shape)} does not fit {kv_heads} key heads of {head_dim}")
    if n * heads >= 1 << 31:
        raise KernelError(f"{n} rows of {heads} heads are too many for one launch")
    return at, n, heads


def page_bounds(keys: torch.Tensor, bounds: torch.Tensor, *, block_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
                max_q_len: int) -> None:
    """Write the bounds of every page that became full in this step: entry ``e`` (a row of ``block_table``) holds ``kv_len[e]``
    tokens now, the last ``q_start[e + 1] - q_start[e]`` of them new.  ``keys`` ``[pages, kv heads, page size, d]``, ``bounds``
    ``[pages, kv heads, 2, d]`` (low, high) of the same type; ``max_q_len``: the most new tokens of an entry (a hint for the
    launch).  Pages that are not full keep what they have; a NaN among a channel's keys makes both bounds NaN."""

    here = native.current_device()
    at = _pool(keys, "keys", here)
    pages, kv_heads, page_size, d = keys.shape
    library = library_name(d)
    _sizes(pages, kv_heads, page_size)
    bounds_at = pointer(bounds, "bounds", here, keys.dtype, shape=(pages, kv_heads, 2, d), align=16)
    kv_len_at = pointer(kv_len, "kv_len", here, torch.int32, dims=1)
    entries = kv_len.shape[0]
    q_start_at = pointer(q_start, "q_start", here, torch.int32, shape=(entries + 1,))
    table_at = pointer(block_table, "block_table", here, torch.int32, dims=2)
    rows, width = block_table.shape
    if rows != entries or (entries and not width):
        raise KernelError(f"a block table of shape {tuple(block_table.shape)} does not fit {entries} entries")
    if max_q_len < 0:
        raise KernelError("max_q_len must not be negative")
    if entries and max_q_len:
        native.call("b200_page_bounds", at, bounds_at, table_at, width, q_start_at, kv_len_at, entries, min(-(-max_q_len // page_size), width), kv_heads,
                    page_size, pages, native.DTYPE_TAG[keys.dtype], stream_ptr(), library=library)


@lru_cache(maxsize=4096)
def choose_shape(rows: int, entries: int, kv_heads: int, width: int, head_dim: int) -> tuple[bool, int]:
    """(tiles of eight rows or not, CTAs of a cluster) of a choice.  Tiles where entries have several rows each, in clusters where the
    scores of many pages want the shared memory or few tiles would not fill the GPU.  For single tokens as many CTAs as let two a
    multiprocessor be there at once, three where each would still have 512 pages (bfloat16, 32 heads over 8 of 128, bounds in L2, clusters of 1, 2, 4
    and 8; 2,048 pages: 1 request 34.5, 21.5, 14.6 and 11.0 us, 8 requests 34.8, 21.9, 17.0 and 22.4, 24 requests 51.6, 41.4, 44.9 and
    59.0, 64 requests 79, 91, 109 and 145; 512 pages: 1 request 12.4, 9.5, 7.8 and 6.7, 24 requests 14.3, 18.5, 21.7 and 33.3)."""

    sms = native.sm_count()
    if rows >= 2 * entries:
        units, sums, cluster = -(-rows // 8) * kv_heads, 2 * head_dim * 64, 1
        while cluster < 8 and sums + 32 * width // cluster > 100 * 1024:
            cluster *= 2
        while cluster < 8 and 2 * cluster * units <= 2 * sms and width // (2 * cluster) >= 64:
            cluster *= 2
        if sums + 32 * width // cluster <= 200 * 1024:
            return True, cluster
    units, cluster = rows * kv_heads, 1
    while cluster < 8 and width // (2 * cluster) >= 64 and 2 * cluster * units <= (3 if width // (2 * cluster) >= 512 else 2) * sms:
        cluster *= 2
    return False, cluster


def choose_pages(q: torch.Tensor, bounds: torch.Tensor, *, positions: torch.Tensor, token_entry: torch.Tensor, block_table: torch.Tensor,
                 page_size: int, budget: int, first: int = 1, last: int = 1) -> torch.Tensor:
    """For every row of ``q`` ``[n, heads, d]`` and every kv head, which of the pages ``0 .. positions[i] // page_size`` of entry
    ``token_entry[i]`` it should read: int32 ``[n, kv heads, budget]``, columns of the block table in rising order, -1 behind
    them.  The ``first`` pages and the ``last`` ones (at least one: the row's own, whose bounds are not up to date) are always
    among them; the others have the highest ``sum over the group's heads and channels of max(q low, q high)``, formed as
    ``sum_c high_c sum_h max(q_hc, 0) + low_c sum_h min(q_hc, 0)`` in 64 bits and rounded to 32; of equal scores the lower page is
    taken, a NaN (an infinite bound that meets a sum of 0 gives one) ranks first.  A page that is not held (an id that is none) is
    not chosen."""

    here = native.current_device()
    at = _pool(bounds, "bounds", here)
    pages, kv_heads, two, d = bounds.shape
    library = library_name(d)
    _sizes(pages, kv_heads)
    if two != 2:
        raise KernelError(f"bounds of shape {tuple(bounds.shape)} are not [pages, kv heads, 2, d]")
    q_at, n, heads = _query(q, kv_heads, d, bounds.dtype, here)
    positions_at, entry_at, table_at, width = _rows(positions, token_entry, block_table, n, here)
    if not 0 < page_size <= MAX_SIZE or first < 0 or last < 1 or not first + last <= budget <= MAX_SIZE:
        raise KernelError(f"page_size {page_size}, budget {budget}, first {first} and last {last}: the budget holds the first pages and "
                          "the last ones, of which there is one at least")
    if width > MAX_TABLE_WIDTH:
        raise KernelError(f"block tables of more than {MAX_TABLE_WIDTH} pages are not taken: {width}")
    chosen = positions.new_empty((n, kv_heads, budget))
    if n:
        entries = block_table.shape[0]
        tiles, cluster = choose_shape(n, entries, kv_heads, width, d)
        native.call("b200_choose_pages_tiles" if tiles else "b200_choose_pages", q_at, at, positions_at, entry_at, table_at, width,
                    chosen.data_ptr(), n, entries, heads, kv_heads, int(page_size), pages, int(budget), int(first), int(last), cluster,
                    native.DTYPE_TAG[bounds.dtype], stream_ptr(), library=library)
    return chosen


@lru_cache(maxsize=4096)
def attention_shape(rows: int, heads: int, kv_heads: int, budget: int, page_size: int, dtype: torch.dtype, head_dim: int = 128) -> tuple[int, bool]:
    """(CTAs of a cluster that the list of a row and kv head is cut over: 1, 2, 4 or 8; twice the warps a CTA).  No part is shorter than
    128 keys.  float32: from the list's length alone, so that the order of the sums does not depend on the batch.  bfloat16: as many
    parts as let two CTAs a multiprocessor be there at once.  A CTA has eight query heads, sixteen of larger groups up to head size 128.
    CTAs of eight heads up to that size have eight warps while the GPU is not full, others always four (2,048 keys a row, parts and "w" for
    eight warps; 32 heads over 8 of 128: 1 request 8: 8.5, 8w: 7.8 us; 8 requests 8: 16.7, 4w: 16.4; 16 requests 2: 30.4, 4: 26.8,
    1w: 29.0, 2w: 26.6; 32 requests 1: 51.6, 2: 48.5, 1w: 46.1, 2w: 51.1; 40 requests 1: 64, 1w: 72, 2w: 72; 64 heads over 4 of 128:
    8 requests 2: 31.1, 4: 19.8, 8: 15.8; 16 requests 1: 46.0, 2: 32.0, 4: 22.6, 8: 30.6; 32 requests 1: 47.4, 2: 36.5, 4: 43.5; 16 heads
    over 4 of 256: 16 requests 2: 34.8, 4: 27.8, 8: 33.7)."""

    keys, parts = budget * page_size, 1
    if dtype == torch.float32:
        while parts < 8 and 2 * parts <= budget and keys // (2 * parts) >= 128:
            parts *= 2
        return parts, False
    group = heads // kv_heads
    ctas = rows * kv_heads * -(-group // (16 if group > 8 and head_dim <= 128 else 8))
    while parts < 8 and 2 * parts <= budget and keys // (2 * parts) >= 128 and 2 * parts * ctas <= 2 * native.sm_count():
        parts *= 2
    return parts, group <= 8 and head_dim <= 128 and ctas * parts <= 2 * native.sm_count()


def paged_attention_chosen(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, chosen: torch.Tensor, *, positions: torch.Tensor,
                           token_entry: torch.Tensor, block_table: torch.Tensor, scale: float) -> torch.Tensor:
    """Attention of row ``i`` of ``q`` ``[n, heads, d]`` over the keys of the pages ``chosen[i, kv head]`` (columns of row
    ``token_entry[i]`` of the block table, distinct, in any order; -1: none) at positions up to ``positions[i]``.  ``keys`` and
    ``values`` are ``[pages, kv heads, page size, d]``.  Keys behind the position and pages that are not held are neither read nor
    counted; a row without a key (or without a score above minus infinity) gives zeros."""

    here = native.current_device()
    at = _pool(keys, "keys", here)
    pages, kv_heads, page_size, d = shape = keys.shape
    library = library_name(d)
    _sizes(pages, kv_heads, page_size)
    values_at = pointer(values, "values", here, keys.dtype, shape=shape, align=16)
    q_at, n, heads = _query(q, kv_heads, d, keys.dtype, here)
    positions_at, entry_at, table_at, width = _rows(positions, token_entry, block_table, n, here)
    chosen_at = pointer(chosen, "chosen", here, torch.int32, dims=3)
    rows, of_heads, budget = chosen.shape
    if rows != n or of_heads != kv_heads or not budget:
        raise KernelError(f"chosen of shape {tuple(chosen.shape)} does not fit {n} rows of {kv_heads} key heads")
    if budget * page_size > MAX_SIZE:
        raise KernelError(f"{budget} pages of {page_size} tokens a row are too many")
    out = torch.empty_like(q)
    if n:
        native.call("b200_attend_chosen", q_at, at, values_at, chosen_at, positions_at, entry_at, table_at, width, out.data_ptr(), n,
                    block_table.shape[0], heads, kv_heads, page_size, pages, budget, float(scale),
                    *attention_shape(n, heads, kv_heads, budget, page_size, keys.dtype, d), native.DTYPE_TAG[keys.dtype], stream_ptr(),
                    library=library)
    return out
