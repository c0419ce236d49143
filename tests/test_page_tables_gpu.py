"""Page tables on the device and the maps of a step, against plain loops over ints."""

import random

import pytest
import torch

from tests.plain import sparse_pages_plain as plain

pytestmark = pytest.mark.gpu


def P():
    from llm_runtime_study_b200.ops import page_tables

    return page_tables


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("rows,width,cells", [(1, 1, 1), (5, 7, 9), (64, 300, 4000)])
def test_set_writes_the_cells_given_and_no_others(rows, width, cells):
    rng = random.Random(rows)
    table = [[rng.randrange(1000) for _ in range(width)] for _ in range(rows)]
    places = rng.sample([(r, c) for r in range(rows) for c in range(width)], cells)
    pages = [rng.randrange(-1, 1 << 30) for _ in places]
    got = ints(table)
    P().page_table_set(got, rows=ints([r for r, _ in places]), columns=ints([c for _, c in places]), pages=ints(pages))
    for (r, c), p in zip(places, pages):
        table[r][c] = p
    assert got.tolist() == table


def test_set_leaves_out_cells_outside_the_table():
    got = torch.zeros((3, 4), dtype=torch.int32, device="cuda")
    room = torch.zeros((5, 4), dtype=torch.int32, device="cuda")
    inner = room[1:4]                         # what lies around it must stay
    cells = [(-1, 0), (3, 0), (0, 4), (2, -1), (1, 2), (2 ** 31 - 1, 2 ** 31 - 1)]
    for t in (got, inner):
        P().page_table_set(t, rows=ints([r for r, _ in cells]), columns=ints([c for _, c in cells]), pages=ints([9] * len(cells)))
    want = torch.zeros((3, 4), dtype=torch.int32)
    want[1, 2] = 9
    assert torch.equal(got.cpu(), want) and torch.equal(room.cpu()[1:4], want) and int(room.sum()) == 9


MAPS = [
    # kv_len, counts, page size, table width
    ([1], [1], 16, 1),
    ([33, 0, 16], [1, 1, 1], 16, 4),
    ([5, 640, 1, 32], [5, 77, 1, 32], 16, 40),
    ([4097, 2500], [4097, 1300], 4, 1026),
    ([300] * 40, [1] * 40, 7, 43),
    ([70, 12], [30, 0], 8, 9),
    ([100], [10], 8, 5),                      # longer than the table is wide
]


@pytest.mark.parametrize("case", MAPS)
@pytest.mark.parametrize("narrow", [False, True])
def test_step_maps(case, narrow):
    kv_len, counts, page, width = case
    rng = random.Random(width)
    rows = len(kv_len) + 2
    tables = [[rng.randrange(10000) for _ in range(width)] for _ in range(rows)]
    tables[0][0] = -1                         # a page given back
    slots = rng.sample(range(rows), len(kv_len))
    n, out_width = sum(counts), max(1, width - 1) if narrow else width
    want = plain.step_maps(tables, slots, kv_len, counts, page, out_width)
    got = P().step_maps(ints(tables), slots=ints(slots), kv_len=ints(kv_len), counts=ints(counts), page_size=page, num_tokens=n,
                        width=out_width if narrow else None)
    assert got.slot_map.dtype == torch.int64
    for name, value in zip(("block_table", "q_start", "positions", "token_entry", "slot_map"), want):
        assert getattr(got, name).tolist() == value, name


def test_slots_outside_the_table_have_no_pages():
    tables = ints([[1, 2], [3, 4]])
    got = P().step_maps(tables, slots=ints([2, -1, 1]), kv_len=ints([20, 20, 20]), counts=ints([1, 2, 1]), page_size=16, num_tokens=4)
    assert got.block_table.tolist() == [[-1, -1], [-1, -1], [3, 4]]
    assert got.slot_map.tolist() == [-1, -1, -1, 4 * 16 + 3] and got.positions.tolist() == [19, 18, 19, 19]


def test_slots_beyond_32_bits():
    tables = ints([[2 ** 30, 2 ** 31 - 1]])
    got = P().step_maps(tables, slots=ints([0]), kv_len=ints([128]), counts=ints([2]), page_size=64, num_tokens=2)
    assert got.slot_map.tolist() == [(2 ** 31 - 1) * 64 + 62, (2 ** 31 - 1) * 64 + 63]


@pytest.mark.parametrize("width", [8, 7])
def test_what_lies_behind_the_last_entry_and_token_stays(width):
    tables = ints([[10 * r + c for c in range(8)] for r in range(4)])

    def full(*shape, dtype=torch.int32):
        return torch.full(shape, 77, dtype=dtype, device="cuda")

    out = P().StepMaps(full(5, width), full(7), full(20), full(20), full(20, dtype=torch.int64))
    got = P().step_maps(tables, slots=ints([3, 1]), kv_len=ints([20, 9]), counts=ints([4, 9]), page_size=4, num_tokens=13, out=out)
    assert got is out
    want = plain.step_maps(tables.tolist(), [3, 1], [20, 9], [4, 9], 4, width)
    for name, value, used in zip(("block_table", "q_start", "positions", "token_entry", "slot_map"), want, (2, 3, 13, 13, 13)):
        t = getattr(out, name)
        assert t[:used].tolist() == value and bool((t[used:] == 77).all()), name
    # tokens beyond what the caller has room for are not written, and what is not wanted is not made
    short = P().StepMaps(full(2, width), None, full(20), None, full(20, dtype=torch.int64))
    P().step_maps(tables, slots=ints([3, 1]), kv_len=ints([20, 9]), counts=ints([4, 9]), page_size=4, num_tokens=6, out=short)
    assert short.positions[:6].tolist() == want[2][:6] and bool((short.positions[6:] == 77).all())
    assert short.slot_map[:6].tolist() == want[4][:6] and bool((short.slot_map[6:] == 77).all())


def test_no_entries():
    got = P().step_maps(ints([[1]]), slots=ints([]), kv_len=ints([]), counts=ints([]), page_size=4, num_tokens=0)
    assert got.block_table.shape == (0, 1) and got.q_start.tolist() == [0] and got.positions.numel() == 0
    P().page_table_set(ints([[1]]), rows=ints([]), columns=ints([]), pages=ints([]))


def test_no_entries_into_tensors_that_are_there():
    def full(*shape, dtype=torch.int32):
        return torch.full(shape, 77, dtype=dtype, device="cuda")

    out = P().StepMaps(full(3, 4), full(4), full(5), full(5), full(5, dtype=torch.int64))
    assert P().step_maps(ints([[1]]), slots=ints([]), kv_len=ints([]), counts=ints([]), page_size=4, num_tokens=0, out=out) is out
    assert out.q_start.tolist() == [0, 77, 77, 77]
    for t in (out.block_table, out.positions, out.token_entry, out.slot_map):
        assert bool((t == 77).all())
