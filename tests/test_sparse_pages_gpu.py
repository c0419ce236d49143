"""Page bounds, the choice of pages and attention over the chosen ones, against plain float64 forms."""

import math

import pytest
import torch

from tests.plain import sparse_pages_plain as plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


def S():
    from llm_runtime_study_b200.ops import sparse_pages

    return sparse_pages


class Cache:
    """Requests of ``lengths`` tokens, the last ``counts`` of them new, in pages of a shuffled pool with spare pages."""

    def __init__(self, lengths, counts, *, heads, kv_heads, d, page, dtype, seed=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.page, self.dtype, self.lengths, self.counts = page, dtype, lengths, counts
        held = [-(-n // page) for n in lengths]
        total, width = sum(held) + spare, max(held + [1]) + 1
        order = torch.randperm(total, generator=g).tolist()
        self.table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        for r, n in enumerate(held):
            self.table[r, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        shape = (total, kv_heads, page, d)
        self.keys, self.values = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
        self.bounds = torch.stack((self.keys.amin(2), self.keys.amax(2)), dim=2)
        n = sum(counts)
        self.q = torch.randn((n, heads, d), generator=g).to(dtype)
        self.positions = torch.cat([torch.arange(a - c, a) for a, c in zip(lengths, counts)]).to(torch.int32)
        self.entry = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(counts)).to(torch.int32)
        self.q_start = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32)
        self.kv_len = torch.tensor(lengths, dtype=torch.int32)

    def rows(self):
        return dict(positions=self.positions.cuda(), token_entry=self.entry.cuda(), block_table=self.table.cuda())

    def choose(self, budget, first=1, last=1):
        return S().choose_pages(self.q.cuda(), self.bounds.cuda(), page_size=self.page, budget=budget, first=first, last=last, **self.rows())

    def plain_choose(self, budget, first=1, last=1):
        return plain.choose_pages(self.q, self.bounds, self.positions, self.entry, self.table, self.page, budget, first, last)

    def attend(self, chosen, scale):
        return S().paged_attention_chosen(self.q.cuda(), self.keys.cuda(), self.values.cuda(), chosen.cuda(), scale=scale, **self.rows())

    def check_attend(self, chosen, scale=None):
        scale = self.q.shape[2] ** -0.5 if scale is None else scale
        got = self.attend(chosen, scale)
        assert got.dtype == self.dtype and got.shape == self.q.shape
        want, size, most, spread = plain.attend_chosen(self.q, self.keys, self.values, chosen.cpu(), self.positions, self.entry,
                                                       self.table, scale)
        off = (got.cpu().double() - want).abs()
        allowed = size * bound(self.dtype, self.q.shape[2], most, spread) + 1e-37
        assert bool((off <= allowed).all()), (float((off / allowed).max()), float(off.max()))
        return got


def bound(dtype, d, keys, spread):
    """How far an output may be off, relative to the weighted sum of |v|.

    A score is a float32 sum of d products of numbers of the type (the scale is one or two roundings more): off by at most
    (d + 3) 2^-24 sum|q k| scale; so is the running maximum's exponent.  A weight exp(s - m) is then off by twice that, by the
    rounding of the exponent's argument (|s - m| <= 2 spread, in units of ln 2) and by 2^-22 of exp itself.  Weights and
    weighted values are summed in float32 over at most ``keys`` terms, and rescaled at most as often.  In bfloat16 the weight
    is rounded once where it meets the value (2^-8), and the output once (2^-8 of its size, at most the weighted |v|)."""

    e = 2.0 ** -24
    score = 2 * (d + 3) * e * spread + 2 * (2 * spread / math.log(2) + 1) * e + 2.0 ** -22
    sums = 2 * (2 * keys + 8) * e
    rounding = 2 * 2.0 ** -8 * (1 + 2.0 ** -7) if dtype == torch.bfloat16 else 2 * e
    return 2 * score + sums + rounding


def some_pages(cache, budget, seed=1, ordered=True):
    """Random distinct pages for every row and kv head, the row's own among them, -1 behind."""

    g = torch.Generator().manual_seed(seed)
    kv_heads = cache.keys.shape[1]
    out = torch.full((cache.q.shape[0], kv_heads, budget), -1, dtype=torch.int32)
    for i in range(cache.q.shape[0]):
        seen = int(cache.positions[i]) // cache.page + 1
        for h in range(kv_heads):
            pages = [seen - 1] + torch.randperm(seen - 1, generator=g)[: budget - 1].tolist() if seen > 1 else [0]
            pages = sorted(pages) if ordered else pages
            out[i, h, : len(pages)] = torch.tensor(pages, dtype=torch.int32)
    return out


# --------------------------------------------------------------------------------------------------------------- bounds
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,kv_heads,page", [(128, 8, 16), (64, 2, 32), (16, 1, 4), (48, 3, 5), (80, 2, 16), (256, 1, 64), (96, 2, 1)])
def test_bounds_of_the_pages_that_became_full(dtype, d, kv_heads, page):
    lengths = [1, page, page + 1, 3 * page, 5 * page - 1, 7 * page + 2, 2 * page]
    counts = [1, 1, 2, 3 * page, 2 * page, 1, page + 1]
    counts = [min(c, n) for c, n in zip(counts, lengths)]
    cache = Cache(lengths, counts, heads=kv_heads, kv_heads=kv_heads, d=d, page=page, dtype=dtype)
    before = torch.full_like(cache.bounds, 7.0)
    want = plain.page_bounds(cache.keys, before, cache.table, lengths, counts)
    assert bool((want != 7).any()) and bool((want == 7).any())
    for hint in (max(counts), 1):           # the hint shapes the launch, not the result
        got = before.cuda()
        S().page_bounds(cache.keys.cuda(), got, block_table=cache.table.cuda(), q_start=cache.q_start.cuda(), kv_len=cache.kv_len.cuda(),
                        max_q_len=hint)
        assert torch.equal(got.cpu(), want)


def test_bounds_skip_pages_that_are_not_held_and_entries_that_are_empty():
    cache = Cache([32, 32, 48, 16], [32, 32, 48, 16], heads=2, kv_heads=2, d=64, page=16, dtype=torch.bfloat16)
    cache.table[1, 0] = -1
    cache.table[2, 1] = 1000                 # not a page of the pool
    cache.kv_len[3] = 0
    before = torch.full_like(cache.bounds, 7.0)
    want = plain.page_bounds(cache.keys, before, cache.table, [32, 32, 48, 0], cache.counts)
    got = before.cuda()
    S().page_bounds(cache.keys.cuda(), got, block_table=cache.table.cuda(), q_start=cache.q_start.cuda(), kv_len=cache.kv_len.cuda(),
                    max_q_len=48)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_bounds_of_nan_and_infinite_keys(dtype):
    cache = Cache([32], [32], heads=1, kv_heads=1, d=64, page=16, dtype=dtype)
    page = int(cache.table[0, 0])
    cache.keys[page, 0, 5, 3] = math.nan
    cache.keys[page, 0, 6, 4] = math.inf
    cache.keys[page, 0, 7, 5] = -math.inf
    got = torch.zeros_like(cache.bounds).cuda()
    S().page_bounds(cache.keys.cuda(), got, block_table=cache.table.cuda(), q_start=cache.q_start.cuda(), kv_len=cache.kv_len.cuda(),
                    max_q_len=32)
    got = got.cpu()
    assert bool(got[page, 0, :, 3].isnan().all())
    assert float(got[page, 0, 1, 4]) == math.inf and float(got[page, 0, 0, 5]) == -math.inf
    want = plain.page_bounds(cache.keys, torch.zeros_like(cache.bounds), cache.table, [32], [32])
    assert torch.equal(got.nan_to_num(9.0), want.nan_to_num(9.0))


# --------------------------------------------------------------------------------------------------------------- choice
CHOICES = [
    # lengths, counts, heads, kv heads, d, page, budget, first, last
    ([1], [1], 4, 1, 64, 16, 4, 1, 1),
    ([37], [1], 8, 2, 64, 4, 3, 1, 2),
    ([700, 33, 64, 129, 1], [1] * 5, 8, 2, 128, 16, 5, 1, 1),
    ([1500, 900], [1, 1], 5, 1, 128, 8, 40, 2, 3),
    ([513], [1], 16, 16, 32, 8, 7, 0, 1),
    ([640, 90, 77], [21, 77, 1], 8, 4, 64, 16, 6, 1, 2),
    ([300, 200], [9, 60], 12, 2, 128, 8, 6, 1, 1),
    ([260], [260], 2, 1, 48, 5, 4, 1, 1),
    ([95], [3], 6, 2, 16, 2, 10, 0, 2),
    ([130], [2], 3, 1, 256, 3, 5, 2, 1),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CHOICES)
def test_chosen_pages(dtype, case):
    lengths, counts, heads, kv_heads, d, page, budget, first, last = case
    cache = Cache(lengths, counts, heads=heads, kv_heads=kv_heads, d=d, page=page, dtype=dtype, seed=len(lengths) + d)
    got = cache.choose(budget, first, last)
    assert got.dtype == torch.int32 and got.shape == (sum(counts), kv_heads, budget)
    assert torch.equal(got.cpu(), cache.plain_choose(budget, first, last))


@pytest.mark.parametrize("rows", [1, 11])
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_chosen_pages_at_every_head_size(dtype, d, rows):
    """Single tokens of several requests, and rows of one."""

    lengths, counts = ([150, 77, 9], [1, 1, 1]) if rows == 1 else ([150], [rows])
    cache = Cache(lengths, counts, heads=6, kv_heads=2, d=d, page=4, dtype=dtype, seed=d)
    assert torch.equal(cache.choose(7, 1, 2).cpu(), cache.plain_choose(7, 1, 2))


@pytest.mark.parametrize("rows", [1, 3])
def test_many_pages(rows):
    """More pages than a CTA has threads many times over, against a vectorised form."""

    d, page, budget, length = 64, 2, 100, 9001
    cache = Cache([length], [rows], heads=2, kv_heads=1, d=d, page=page, dtype=torch.bfloat16)
    x = cache.q.double()
    b = cache.bounds[cache.table[0, : -(-length // page)].long(), 0].double()
    score = (x.clamp(min=0).sum(1) @ b[:, 1].T + x.clamp(max=0).sum(1) @ b[:, 0].T).float()
    got = cache.choose(budget, 2, 3).cpu()
    for i in range(rows):
        seen = int(cache.positions[i]) // page + 1
        order = score[i, 2 : seen - 3].argsort(descending=True, stable=True)[: budget - 5] + 2
        want = torch.cat((torch.tensor([0, 1]), order.sort().values, torch.arange(seen - 3, seen)))
        assert torch.equal(got[i, 0].long(), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_head_sizes_one_after_the_other_in_one_process(dtype):
    """Every head size is a library of its own, and each has to raise its kernels' limit of shared memory: the scores of 13,000 pages
    are more than a kernel gets unasked."""

    for d in (64, 128, 32, 256, 16):
        for length, rows in ((13000, 8), (13000, 1)):
            cache = Cache([length], [rows], heads=2, kv_heads=1, d=d, page=1, dtype=dtype, seed=d)
            got = cache.choose(40, 1, 2).cpu()
            x = cache.q.double()
            b = cache.bounds[cache.table[0, :length].long(), 0].double()
            score = (x.clamp(min=0).sum(1) @ b[:, 1].T + x.clamp(max=0).sum(1) @ b[:, 0].T).float()
            for i in range(rows):
                seen = int(cache.positions[i]) + 1
                order = score[i, 1 : seen - 2].argsort(descending=True, stable=True)[:37] + 1
                want = torch.cat((torch.tensor([0]), order.sort().values, torch.arange(seen - 2, seen)))
                assert torch.equal(got[i, 0].long(), want), (d, length)


@pytest.mark.parametrize("rows", [1, 12])
@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_scores_go_to_the_lower_page(dtype, rows):
    cache = Cache([400], [rows], heads=4, kv_heads=2, d=64, page=8, dtype=dtype)
    cache.bounds[:] = cache.bounds[0]                        # every page alike
    got = cache.choose(9, 1, 2).cpu()
    for i in range(rows):
        seen = int(cache.positions[i]) // 8 + 1
        assert got[i, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, seen - 2, seen - 1]
    cache.bounds[:] = 0.0                                    # and zeros of either sign
    cache.bounds[::2, :, 0] = -0.0
    assert torch.equal(cache.choose(9, 1, 2).cpu(), got)
    assert torch.equal(cache.plain_choose(9, 1, 2), got)


@pytest.mark.parametrize("rows", [1, 12])
@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_that_differ_in_their_last_bits(dtype, d, rows):
    """Pages alike but for one small channel, one step up or down: scores a few float32 steps apart, or equal."""

    cache = Cache([600], [rows], heads=4, kv_heads=2, d=d, page=4, dtype=dtype, seed=d)
    g = torch.Generator().manual_seed(5)
    cache.bounds[:] = cache.bounds[0]
    channel = int(cache.q[0].float().abs().sum(0).argmin())
    step = torch.finfo(dtype).eps * torch.randint(-3, 4, (cache.bounds.shape[0], 2, 2), generator=g)
    cache.bounds[..., channel] = (cache.bounds[..., channel].float() * (1 + step)).to(dtype)
    for budget in (5, 20, 75):
        assert torch.equal(cache.choose(budget, 1, 2).cpu(), cache.plain_choose(budget, 1, 2))


@pytest.mark.parametrize("rows", [1, 10])
@pytest.mark.parametrize("q_scale,bound_scale", [(1e-30, 1.0), (1e-36, 1e-5), (1e-38, 1e30), (1e30, 1e-30), (1e18, 1e18), (1.0, 1e38), (0.0, 1.0), (1.0, 1e-39)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_very_small_and_very_large_numbers(dtype, q_scale, bound_scale, rows):
    cache = Cache([300], [rows], heads=4, kv_heads=2, d=32, page=4, dtype=dtype)
    cache.q = (cache.q.double() * q_scale).to(dtype)
    cache.bounds = (cache.bounds.double() * bound_scale).to(dtype)
    assert torch.equal(cache.choose(20, 1, 2).cpu(), cache.plain_choose(20, 1, 2))


@pytest.mark.parametrize("rows", [1, 9])
@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_ranks_first_and_infinities_keep_their_order(dtype, rows):
    cache = Cache([320], [rows], heads=2, kv_heads=2, d=32, page=8, dtype=dtype)
    cache.q[:] = cache.q.abs() + 0.5                         # every head looks at the upper bounds
    at = cache.table[0].long()
    cache.bounds[at[:40], :, 0] = 0.0
    cache.bounds[at[:40], :, 1] = cache.bounds[at[:40], :, 1].clamp(max=3)
    cache.bounds[at[20], 0, 1, 3] = math.nan
    cache.bounds[at[25], 0, 1, 4] = math.inf
    cache.bounds[at[30], 1, :, 5] = -math.inf               # no head looks down: 0 times infinity
    for budget in (3, 4, 10, 37):
        got = cache.choose(budget, 1, 1).cpu()
        assert torch.equal(got, cache.plain_choose(budget, 1, 1))
        assert bool((got[:, 0] == 20).any(-1).all())
        assert bool((got[:, 0] == 25).any(-1).all()) == (budget >= 4)
        assert bool((got[:, 1] == 30).any(-1).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_stand_nowhere_and_pages_that_are_not_held(dtype):
    cache = Cache([200, 160, 96, 64, 40, 90], [1] * 6, heads=4, kv_heads=2, d=64, page=8, dtype=dtype)
    cache.table[1] = -1                       # a row that pads the batch
    cache.table[0, 3:9] = -1                  # pages given back
    cache.table[2, 5] = 10_000                # not a page of the pool
    cache.positions[3] = -1
    cache.entry[4] = 17
    cache.positions[5] = 10_000               # behind the table: its last columns
    for budget in (3, 6, 30):
        got = cache.choose(budget, 1, 1)
        assert torch.equal(got.cpu(), cache.plain_choose(budget, 1, 1))
        assert bool((got[1] == -1).all()) and bool((got[3] == -1).all()) and bool((got[4] == -1).all())
        out = cache.check_attend(got)
        assert float(out[[1, 3, 4]].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_last_position_there_is(dtype):
    """Pages of one token: a page's number and the count of pages up to it are 32-bit numbers, and the count must not wrap."""

    cache = Cache([70, 70, 70, 70], [1, 1, 1, 1], heads=4, kv_heads=2, d=64, page=1, dtype=dtype)
    cache.positions[1] = 2 ** 31 - 1
    cache.positions[2] = 2 ** 31 - 2
    for budget in (5, 100):
        got = cache.choose(budget, 1, 2)
        assert torch.equal(got.cpu(), cache.plain_choose(budget, 1, 2))
        assert bool((got[1] >= 0).any())
        cache.check_attend(got)


# ------------------------------------------------------------------------------------------------------------ attention
ATTENTION = [
    # lengths, counts, heads, kv heads, d, page, budget
    ([1], [1], 4, 1, 64, 16, 4),
    ([16], [1], 1, 1, 128, 16, 1),
    ([700, 33, 64, 129, 1], [1] * 5, 8, 2, 128, 16, 5),
    ([2500, 37], [1, 1], 8, 1, 128, 16, 128),
    ([513, 400], [1, 1], 5, 1, 64, 32, 7),
    ([640, 90], [21, 40], 12, 4, 64, 16, 6),
    ([300], [7], 18, 2, 128, 64, 4),
    ([300], [3], 20, 1, 32, 16, 9),
    ([260], [30], 2, 1, 48, 5, 20),
    ([95], [3], 6, 2, 16, 2, 10),
    ([130], [2], 3, 1, 256, 3, 33),
    ([222, 99], [5, 1], 7, 7, 80, 8, 11),
    ([150], [2], 34, 2, 96, 16, 8),
    ([400], [1], 16, 2, 112, 24, 9),
    ([5000], [1], 16, 2, 64, 4, 600),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ATTENTION)
def test_attention_over_chosen_pages(dtype, case):
    lengths, counts, heads, kv_heads, d, page, budget = case
    cache = Cache(lengths, counts, heads=heads, kv_heads=kv_heads, d=d, page=page, dtype=dtype, seed=d + heads)
    chosen = some_pages(cache, budget)
    out = cache.check_attend(chosen)
    # the order of the list does not matter beyond the order of the sums
    other = cache.attend(some_pages(cache, budget, ordered=False), d ** -0.5)
    torch.testing.assert_close(other.float(), out.float(), atol=2e-2 if dtype == torch.bfloat16 else 2e-5, rtol=0)


LONG_LISTS = [
    # length, rows, heads, kv heads, d, page, budget
    (5000, 1, 4, 2, 64, 1, 4400),
    (9100, 1, 16, 1, 48, 2, 4500),                # 16 heads in bfloat16: two tiles of heads a CTA
    (4200 * 16 + 5, 1, 2, 1, 64, 16, 4150),       # whole tiles
    (1300, 80, 4, 2, 16, 1, 1100),                # bfloat16: rows enough for lists that are not cut, three laps
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", LONG_LISTS)
def test_lists_longer_than_a_cta_looks_up_at_a_time(dtype, case):
    """A CTA looks up 512 pages of its part of a list at a time and comes back for more."""

    length, rows, heads, kv_heads, d, page, budget = case
    parts, _ = S().attention_shape(rows, heads, kv_heads, budget, page, dtype)
    laps = -(-budget // parts // 512)
    assert laps >= (3 if rows > 1 and dtype == torch.bfloat16 else 1 if rows > 1 else 2)
    cache = Cache([length], [rows], heads=heads, kv_heads=kv_heads, d=d, page=page, dtype=dtype, seed=budget)
    chosen = some_pages(cache, budget)
    cache.check_attend(chosen)
    # a list whose later laps alone hold anything
    late = chosen.clone()
    late[:, :, : 512 * parts] = -1
    if laps > 1:
        assert bool((late >= 0).any(-1).all())
        cache.check_attend(late)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores_and_one_heavy_key(dtype):
    cache = Cache([700, 300], [1, 4], heads=8, kv_heads=2, d=64, page=16, dtype=dtype)
    cache.q *= 6
    cache.check_attend(some_pages(cache, 20))
    cache.check_attend(some_pages(cache, 20), scale=-0.7)
    cache.check_attend(some_pages(cache, 20), scale=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 4, 24])
def test_what_a_mask_hides_is_not_read(dtype, page):
    """NaN and infinities behind the row's position, on pages not chosen and on pages of nobody."""

    cache = Cache([5 * page + 3, 3 * page, 1], [1, 1, 1], heads=4, kv_heads=2, d=64, page=page, dtype=dtype)
    chosen = some_pages(cache, 3)
    want = cache.check_attend(chosen)
    for t in (cache.keys, cache.values):
        for r, length in enumerate(cache.lengths):
            for c in range(cache.table.shape[1]):
                p = int(cache.table[r, c])
                if p < 0:
                    continue
                for h in range(2):
                    if c not in chosen[r, h].tolist():
                        t[p, h] = math.nan
                    elif (c + 1) * page > length:
                        t[p, h, length - c * page :] = math.inf if t is cache.keys else math.nan
        for p in set(range(t.shape[0])) - set(cache.table.flatten().tolist()):
            t[p] = math.nan
    assert torch.equal(cache.attend(chosen, 64 ** -0.5), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lists_with_holes_and_pages_that_are_none(dtype):
    cache = Cache([200, 120], [1, 6], heads=4, kv_heads=2, d=64, page=16, dtype=dtype)
    chosen = some_pages(cache, 12)
    chosen[:, :, 3] = -1
    chosen[0, 1, 5] = 999                     # behind the table
    chosen[2, 0] = -1                         # nothing at all
    chosen[3, 1, -1] = 11                     # a page the request does not hold
    cache.table[1, 2] = -1
    cache.table[0, 4] = 12345                 # not a page of the pool
    out = cache.check_attend(chosen)
    assert float(out[2, :2].abs().max()) == 0.0


def test_a_pool_that_needs_more_than_32_bits_of_offset():
    """Pages whose elements lie beyond 2^31 of the pool's start."""

    page, kv_heads, d = 64, 8, 128
    pages = (1 << 31) // (page * kv_heads * d) + 40
    keys = torch.zeros((pages, kv_heads, page, d), dtype=torch.bfloat16, device="cuda")
    values = torch.zeros_like(keys)
    bounds = torch.zeros((pages, kv_heads, 2, d), dtype=torch.bfloat16, device="cuda")
    ids = [pages - 1, 3, pages - 7, pages - 20, 11, pages - 30]
    small = Cache([6 * page], [1], heads=16, kv_heads=kv_heads, d=d, page=page, dtype=torch.bfloat16, spare=0)
    for c, p in enumerate(ids):
        keys[p] = small.keys[int(small.table[0, c])].cuda()
        values[p] = small.values[int(small.table[0, c])].cuda()
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    rows = dict(positions=small.positions.cuda(), token_entry=small.entry.cuda(), block_table=table)
    for length in range(page, 7 * page, page):
        S().page_bounds(keys, bounds, block_table=table, q_start=small.q_start.cuda(),
                        kv_len=torch.tensor([length], dtype=torch.int32, device="cuda"), max_q_len=1)
    for c, p in enumerate(ids):
        assert torch.equal(bounds[p].cpu(), small.bounds[int(small.table[0, c])])
    chosen = S().choose_pages(small.q.cuda(), bounds, page_size=page, budget=4, **rows)
    assert torch.equal(chosen, small.choose(4))
    out = S().paged_attention_chosen(small.q.cuda(), keys, values, chosen, scale=0.1, **rows)
    assert torch.equal(out, small.attend(chosen, 0.1))


@pytest.mark.parametrize("tail", [16, 8])         # whole tiles of 16 keys, and a page that ends inside one
def test_a_page_that_needs_more_than_32_bits_of_offset(tail):
    """One page of more than 2^31 elements: keys that matter in front of that border, at it and behind it.  Those three have the same
    score, 40 above every other key's, so the row is the mean of their values: 2^24 others weigh 2^24 e^-40 = 7e-11 in all and have
    values of zero, equal weights are exactly one in bfloat16, so that the rounding of the output (2^-8) is all that is off."""

    d, border = 128, (1 << 31) // 128
    page = border + tail
    keys, values = (torch.zeros((1, 1, page, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(tail)
    heavy = torch.randn((3, d), generator=g).to(torch.bfloat16)
    for at, v in zip((3, border - 1, border + 5), heavy):
        keys[0, 0, at, 0] = 5.0
        values[0, 0, at] = v.cuda()
    q = torch.zeros((1, 2, d), dtype=torch.bfloat16, device="cuda")
    q[:, :, 0] = 8.0
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")      # noqa: E731
    rows = dict(token_entry=ints(0), block_table=ints([0]), scale=1.0)
    for position, seen in ((page - 1, 3), (border + 5, 3), (border + 4, 2), (border - 2, 1)):
        out = S().paged_attention_chosen(q, keys, values, ints([[0]]), positions=ints(position), **rows)
        want = heavy[:seen].double().mean(0)
        assert bool(((out.cpu().double() - want).abs() <= want.abs() * 2.0 ** -8 + 1e-6).all()), position


# ------------------------------------------------------------------------------------------------------------- together
def _layer(cache, keys, values, bounds, q, positions, entry, table, q_start, kv_len, budget):
    S().page_bounds(keys, bounds, block_table=table, q_start=q_start, kv_len=kv_len, max_q_len=q.shape[0])
    rows = dict(positions=positions, token_entry=entry, block_table=table)
    chosen = S().choose_pages(q, bounds, page_size=cache.page, budget=budget, first=1, last=2, **rows)
    return chosen, S().paged_attention_chosen(q, keys, values, chosen, scale=0.125, **rows)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_sequence_in_portions_and_token_by_token_gives_the_same_rows(dtype):
    """Bounds, choice and attention over a growing cache: one portion, several, single tokens."""

    cache = Cache([230], [230], heads=4, kv_heads=2, d=64, page=8, dtype=dtype)
    q, table = cache.q.cuda(), cache.table.cuda()
    results = []
    for cuts in ([230], [1, 7, 8, 100, 114], [1] * 230):
        # the pages fill up as the tokens come: what lies behind a portion is not there yet
        keys, values = (torch.full_like(t, math.nan).cuda() for t in (cache.keys, cache.values))
        bounds = torch.full_like(cache.bounds, math.nan).cuda()
        chosen, out, at = [], [], 0
        for n in cuts:
            for p in range(at, at + n):
                for pool, source in ((keys, cache.keys), (values, cache.values)):
                    pool[int(cache.table[0, p // 8]), :, p % 8] = source[int(cache.table[0, p // 8]), :, p % 8].cuda()
            ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, n], [at + n])]
            c, o = _layer(cache, keys, values, bounds, q[at : at + n], torch.arange(at, at + n, dtype=torch.int32, device="cuda"),
                          torch.zeros(n, dtype=torch.int32, device="cuda"), table, *ints, 6)
            chosen.append(c)
            out.append(o)
            at += n
        results.append((torch.cat(chosen), torch.cat(out)))
    assert torch.equal(results[0][0].cpu(), cache.plain_choose(6, 1, 2))
    cache.check_attend(results[0][0], scale=0.125)
    for chosen, out in results[1:]:
        assert torch.equal(chosen, results[0][0])
        if dtype == torch.float32:
            assert torch.equal(out, results[0][1])
        else:
            torch.testing.assert_close(out.float(), results[0][1].float(), atol=2e-2, rtol=0)


def test_captured_and_replayed_with_other_lengths_and_inputs():
    cache = Cache([250, 90, 17], [1, 1, 1], heads=8, kv_heads=2, d=64, page=8, dtype=torch.bfloat16, seed=3)
    other = Cache([250, 90, 17], [1, 1, 1], heads=8, kv_heads=2, d=64, page=8, dtype=torch.bfloat16, seed=4)
    names = ("keys", "values", "bounds", "q", "positions", "entry", "table", "q_start", "kv_len")
    held = {n: getattr(cache, n).cuda() for n in names}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _layer(cache, *[held[n] for n in names], 6)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chosen, out = _layer(cache, *[held[n] for n in names], 6)
    other.kv_len[1] = 40                      # a shorter sequence, and a row that pads the batch
    other.positions[1] = 39
    other.kv_len[2], other.positions[2] = 0, 0
    other.table[2] = -1
    for source in (cache, other, cache):
        for n in names:
            held[n].copy_(getattr(source, n))
        graph.replay()
        fresh = {n: getattr(source, n).cuda() for n in names}
        want = _layer(source, *[fresh[n] for n in names], 6)
        assert torch.equal(chosen, want[0]) and torch.equal(out, want[1])
        assert torch.equal(chosen.cpu(), source.plain_choose(6, 1, 2))
    assert float(out[2].abs().max()) > 0


def test_two_streams_at_once():
    cases = [Cache([900, 333], [1, 1], heads=8, kv_heads=2, d=128, page=16, dtype=torch.bfloat16, seed=s) for s in (1, 2)]
    wants = [(c.choose(9), c.attend(some_pages(c, 9), 0.1)) for c in cases]
    held = [(c.q.cuda(), c.bounds.cuda(), c.keys.cuda(), c.values.cuda(), some_pages(c, 9).cuda(), c.rows()) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (q, bounds, keys, values, pages, rows) in enumerate(held):
            with torch.cuda.stream(streams[i]):
                got[i].append((S().choose_pages(q, bounds, page_size=16, budget=9, **rows),
                               S().paged_attention_chosen(q, keys, values, pages, scale=0.1, **rows)))
    torch.cuda.synchronize()
    for want, runs in zip(wants, got):
        for chosen, out in runs:
            assert torch.equal(chosen, want[0]) and torch.equal(out, want[1])
