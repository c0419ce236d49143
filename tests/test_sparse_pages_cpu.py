"""What the page-table and chosen-page operators refuse, on the host and before anything is launched; their plain forms."""

import math

import pytest
import torch

from llm_runtime_study_b200.errors import KernelError
from llm_runtime_study_b200.ops import native, page_tables, sparse_pages
from tests.plain import sparse_pages_plain as plain


@pytest.fixture
def host(monkeypatch):
    """The operators with CPU tensors taken for CUDA ones; a launch is an error of the test."""

    def pointer(t, name, here, dtype, shape=None, dims=None, align=4):
        if t.dtype is not dtype or not t.is_contiguous() or (shape is not None and t.shape != shape) or (dims is not None and t.dim() != dims):
            raise KernelError(name)
        if t.data_ptr() % align:
            raise KernelError(f"{name} must start on a multiple of {align} bytes")
        return t.data_ptr()

    def require(t, name, *, dtype=None, **_):
        if t.dtype not in (dtype if isinstance(dtype, (tuple, list)) else (dtype,)):
            raise KernelError(f"{name} has dtype {t.dtype}")

    launched = []
    for module in (page_tables, sparse_pages):
        monkeypatch.setattr(module, "pointer", pointer)
    monkeypatch.setattr(native, "require", require)
    for module in (native, sparse_pages):
        monkeypatch.setattr(module, "stream_ptr", lambda: 0)
    monkeypatch.setattr(native, "call", lambda *a, **k: launched.append(a[0]))
    return launched


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def good():
    return dict(q=torch.zeros(3, 4, 64), keys=torch.zeros(5, 2, 8, 64), values=torch.zeros(5, 2, 8, 64), bounds=torch.zeros(5, 2, 2, 64),
                chosen=ints(3, 2, 6), positions=ints(3), token_entry=ints(3), block_table=ints(2, 9), q_start=ints(3), kv_len=ints(2))


def _bounds(a):
    sparse_pages.page_bounds(a["keys"], a["bounds"], block_table=a["block_table"], q_start=a["q_start"], kv_len=a["kv_len"],
                             max_q_len=a.get("max_q_len", 2))


def _choose(a):
    return sparse_pages.choose_pages(a["q"], a["bounds"], positions=a["positions"], token_entry=a["token_entry"],
                                     block_table=a["block_table"], page_size=a.get("page_size", 8), budget=a.get("budget", 4),
                                     first=a.get("first", 1), last=a.get("last", 1))


def _attend(a):
    return sparse_pages.paged_attention_chosen(a["q"], a["keys"], a["values"], a["chosen"], positions=a["positions"],
                                               token_entry=a["token_entry"], block_table=a["block_table"], scale=0.1)


def test_good_arguments_are_launched(host):
    _bounds(good())
    assert _choose(good()).shape == (3, 2, 4)
    assert _attend(good()).shape == (3, 4, 64)
    assert host == ["b200_page_bounds", "b200_choose_pages", "b200_attend_chosen"]
    empty = good() | dict(q=torch.zeros(0, 4, 64), chosen=ints(0, 2, 6), positions=ints(0), token_entry=ints(0))
    assert _choose(empty).shape == (0, 2, 4) and _attend(empty).shape == (0, 4, 64)
    _bounds(good() | dict(max_q_len=0))
    assert len(host) == 3                     # nothing to do is nothing launched


MISALIGNED = torch.zeros(3 * 4 * 64 + 1)[1:].view(3, 4, 64)
REFUSED = [
    (_bounds, dict(keys=torch.zeros(5, 2, 8, 24), bounds=torch.zeros(5, 2, 2, 24))),
    (_bounds, dict(keys=torch.zeros(5, 2, 8, 272), bounds=torch.zeros(5, 2, 2, 272))),
    (_bounds, dict(keys=torch.zeros(5, 2, 8, 64, dtype=torch.float16))),
    (_bounds, dict(keys=torch.zeros(0, 2, 8, 64), bounds=torch.zeros(0, 2, 2, 64))),
    (_bounds, dict(bounds=torch.zeros(5, 2, 2, 64, dtype=torch.bfloat16))),
    (_bounds, dict(bounds=torch.zeros(5, 2, 64))),
    (_bounds, dict(bounds=torch.zeros(4, 2, 2, 64))),
    (_bounds, dict(kv_len=ints(3))),
    (_bounds, dict(kv_len=ints(2).long())),
    (_bounds, dict(q_start=ints(2))),
    (_bounds, dict(block_table=ints(3, 9))),
    (_bounds, dict(block_table=ints(2, 0))),
    (_bounds, dict(max_q_len=-1)),
    (_bounds, dict(keys=torch.zeros(5, 8, 2, 64).transpose(1, 2))),
    (_choose, dict(q=torch.zeros(3, 5, 64))),
    (_choose, dict(q=torch.zeros(3, 0, 64))),
    (_choose, dict(q=torch.zeros(3, 4, 32))),
    (_choose, dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16))),
    (_choose, dict(q=torch.zeros(4, 3, 64).transpose(0, 1))),
    (_choose, dict(q=MISALIGNED)),
    (_choose, dict(bounds=torch.zeros(5, 2, 3, 64))),
    (_choose, dict(positions=ints(2))),
    (_choose, dict(token_entry=ints(4))),
    (_choose, dict(positions=ints(3).long())),
    (_choose, dict(block_table=ints(9))),
    (_choose, dict(block_table=ints(0, 9))),
    (_choose, dict(block_table=ints(2, sparse_pages.MAX_TABLE_WIDTH + 1))),
    (_choose, dict(page_size=0)),
    (_choose, dict(page_size=(1 << 32) + 16)),
    (_choose, dict(budget=1 << 31)),
    (_choose, dict(budget=1)),
    (_choose, dict(budget=3, first=2, last=2)),
    (_choose, dict(last=0)),
    (_choose, dict(first=-1)),
    (_attend, dict(values=torch.zeros(5, 2, 8, 32))),
    (_attend, dict(values=torch.zeros(5, 2, 8, 64, dtype=torch.bfloat16))),
    (_attend, dict(chosen=ints(3, 1, 6))),
    (_attend, dict(chosen=ints(2, 2, 6))),
    (_attend, dict(chosen=ints(3, 2, 0))),
    (_attend, dict(chosen=ints(3, 2, 6).long())),
    (_attend, dict(q=MISALIGNED)),
    (_attend, dict(keys=torch.zeros(5, 3, 8, 64), values=torch.zeros(5, 3, 8, 64))),
    (_attend, dict(positions=ints(4))),
]


@pytest.mark.parametrize("at", range(len(REFUSED)))
def test_what_does_not_fit_is_refused_before_a_launch(host, at):
    call, change = REFUSED[at]
    with pytest.raises(KernelError):
        call(good() | change)
    assert host == []


def test_page_tables_refuse_what_does_not_fit(host):
    tables = ints(3, 4)

    def maps(**change):
        given = dict(slots=ints(2), kv_len=ints(2), counts=ints(2), page_size=8, num_tokens=4) | change
        return page_tables.step_maps(given.pop("tables", tables), **given)

    assert maps().block_table.shape == (2, 4) and maps(width=2).block_table.shape == (2, 2)
    assert host == ["b200_step_maps"] * 2
    host.clear()
    made = page_tables.StepMaps(ints(2, 4), ints(3), ints(4), ints(4), ints(4).long())
    for change in (dict(tables=ints(3)), dict(tables=ints(0, 4)), dict(tables=tables.long()), dict(slots=ints(3)), dict(counts=ints(1)),
                   dict(kv_len=ints(2).long()), dict(page_size=0), dict(page_size=(1 << 32) + 8), dict(num_tokens=1 << 32), dict(width=1 << 32),
                   dict(num_tokens=-1), dict(width=0), dict(width=3, out=made),
                   dict(num_tokens=5, out=made), dict(tables=ints(4, 3).T)):
        with pytest.raises(KernelError):
            maps(**change)
    for name, value in (("block_table", ints(1, 4)), ("block_table", ints(8)), ("q_start", ints(2)), ("positions", ints(4).long()),
                        ("token_entry", ints(3)), ("slot_map", ints(4))):
        out = page_tables.StepMaps(**(vars(made) | {name: value}))
        with pytest.raises(KernelError):
            maps(out=out)
    for change in (dict(tables=ints(0, 0)), dict(columns=ints(1)), dict(pages=ints(2).long()), dict(rows=ints(2, 1))):
        given = dict(rows=ints(2), columns=ints(2), pages=ints(2)) | change
        with pytest.raises(KernelError):
            page_tables.page_table_set(given.pop("tables", tables), **given)
    assert host == []


def test_cpu_tensors_are_refused():
    for call in (_bounds, _choose, _attend):
        with pytest.raises(KernelError, match="CUDA"):
            call(good())
    with pytest.raises(KernelError, match="CUDA"):
        page_tables.page_table_set(ints(3, 4), rows=ints(1), columns=ints(1), pages=ints(1))
    with pytest.raises(KernelError, match="CUDA"):
        page_tables.step_maps(ints(3, 4), slots=ints(1), kv_len=ints(1), counts=ints(1), page_size=8, num_tokens=1)


def test_tensors_of_another_device_are_refused():
    class Elsewhere(torch.Tensor):
        is_cuda, index = True, 1
        device = torch.device("cuda", 1)

        def get_device(self):
            return self.index

    t = torch.zeros(64, dtype=torch.int32).as_subclass(Elsewhere)
    with pytest.raises(KernelError, match="current device"):
        native.pointer(t, "q", 0, torch.int32)
    Elsewhere.index = 0
    assert native.pointer(t, "q", 0, torch.int32, shape=(64,), dims=1) == t.data_ptr()
    for wrong in (dict(shape=(63,)), dict(dims=2)):
        with pytest.raises(KernelError):
            native.pointer(t, "q", 0, torch.int32, **wrong)
    for wrong in (None, 7, "q"):
        with pytest.raises(KernelError, match="CUDA"):
            native.pointer(wrong, "q", 0, torch.int32)
    with pytest.raises(KernelError, match="dtype"):
        native.pointer(t, "q", 0, torch.int64)
    with pytest.raises(KernelError, match="multiple"):
        native.pointer(t[1:], "q", 0, torch.int32, align=16)


def test_a_page_s_score_bounds_the_scores_of_its_keys():
    g = torch.Generator().manual_seed(0)
    keys = torch.randn(6, 1, 8, 16, generator=g, dtype=torch.float64)
    q = torch.randn(1, 3, 16, generator=g, dtype=torch.float64)
    low, high = keys.amin(2), keys.amax(2)
    score = torch.maximum(q[0, :, None] * low[:, 0], q[0, :, None] * high[:, 0]).sum(-1)
    assert bool((score[:, :, None] >= torch.einsum("hd,psd->hps", q[0], keys[:, 0]) - 1e-12).all())
    together = high[:, 0] @ q[0].clamp(min=0).sum(0) + low[:, 0] @ q[0].clamp(max=0).sum(0)
    torch.testing.assert_close(together, score.sum(0))
    assert not math.isnan(float(score.sum()))


def test_plain_choice_keeps_the_first_and_the_last_pages():
    q, bounds = torch.ones(1, 1, 16), torch.zeros(9, 1, 2, 16)
    bounds[4, 0, 1] = 5.0
    table = torch.arange(9, dtype=torch.int32)[None]
    at = torch.tensor([70]), torch.tensor([0])
    assert plain.choose_pages(q, bounds, *at, table, 8, 4, 1, 2).tolist() == [[[0, 4, 7, 8]]]
    assert plain.choose_pages(q, bounds, *at, table, 8, 5, 1, 2).tolist() == [[[0, 1, 4, 7, 8]]]


def test_shapes_of_the_launches():
    """On a B200's 148 multiprocessors (what the rules assume where no device is visible)."""

    shape = lambda *a: sparse_pages.choose_shape.__wrapped__(*a)      # noqa: E731
    assert [shape(n, n, 8, 2048, 128) for n in (1, 8, 16, 24, 64)] == [(False, c) for c in (8, 4, 2, 2, 1)]
    assert [shape(n, n, 8, 512, 128) for n in (1, 24)] == [(False, 8), (False, 1)]
    assert shape(1, 1, 1, 4, 64) == (False, 1)
    assert shape(500, 2, 8, 1024, 128) == (True, 1) and shape(8, 1, 1, 1024, 128) == (True, 8)
    assert shape(500, 2, 8, 8192, 128)[0] and shape(500, 2, 8, 8192, 128)[1] >= 4       # scores of many pages lie in several CTAs
    for width in (1, 100, 3000, 20000, sparse_pages.MAX_TABLE_WIDTH):                    # and what is chosen fits
        for d in (16, 128, 256):
            for rows, entries in ((1, 1), (40, 1), (40, 40)):
                tiles, cluster = shape(rows, entries, 8, width, d)
                assert cluster in (1, 2, 4, 8)
                assert (width * (8 // cluster) * 4 + 2 * d * 64 if tiles else width * 4) <= 200 * 1024
    attend = lambda *a: sparse_pages.attention_shape.__wrapped__(*a)      # noqa: E731
    bf16, f32 = torch.bfloat16, torch.float32
    assert [attend(n, 32, 8, 128, 16, bf16) for n in (1, 8, 16, 24, 40)] == [(8, True), (4, True), (2, True), (1, True), (1, False)]
    assert attend(1, 32, 8, 4, 16, bf16) == (1, True) and attend(1, 8, 8, 1, 4096, bf16) == (1, True)      # one page is one part
    assert attend(1, 32, 8, 128, 16, f32) == attend(4000, 32, 8, 128, 16, f32) == (8, False)               # the list alone decides


def test_shapes_count_the_ctas_that_are_launched():
    """Groups of more than eight heads: sixteen a CTA up to head size 128, and no CTAs of eight warps; none at larger head sizes."""

    attend = lambda n, heads, kv_heads, d: sparse_pages.attention_shape.__wrapped__(n, heads, kv_heads, 128, 16, torch.bfloat16, d)      # noqa: E731
    assert [attend(n, 64, 4, 128) for n in (1, 8, 12, 16, 32, 48)] == [(p, False) for p in (8, 8, 4, 4, 2, 1)]
    assert [attend(n, 96, 8, 64) for n in (4, 8, 16, 24)] == [(p, False) for p in (8, 4, 2, 1)]
    assert [attend(n, 96, 4, 128) for n in (4, 16, 32)] == [(p, False) for p in (8, 2, 1)]       # 24 heads a group: two CTAs
    assert [attend(n, 16, 4, 256) for n in (8, 16, 32)] == [(p, False) for p in (8, 4, 2)]
    assert [attend(n, 64, 4, 256) for n in (8, 16, 32)] == [(p, False) for p in (4, 2, 1)]       # 16 heads a group: two CTAs there
    assert attend(8, 32, 8, 128) == (4, True)


@pytest.mark.parametrize("max_seq_len,pages,want", [(400, 10, 10), (400, 10 ** 9, 25), (400, 25, 25), (20, 10 ** 9, 3), (20, 3, 3)])
def test_a_layer_asks_for_no_more_pages_than_a_sequence_has(monkeypatch, max_seq_len, pages, want):
    from types import SimpleNamespace

    from llm_runtime_study_b200.parts.attention import GroupedQueryAttention

    asked = []
    monkeypatch.setattr(sparse_pages, "page_bounds", lambda *a, **k: None)
    monkeypatch.setattr(sparse_pages, "choose_pages", lambda *a, budget, **k: asked.append(budget))
    monkeypatch.setattr(sparse_pages, "paged_attention_chosen", lambda q, *a, **k: q)
    pool = SimpleNamespace(pages_for=lambda n: -(-n // 16))
    ctx = SimpleNamespace(manager=SimpleNamespace(groups=[pool], max_seq_len=max_seq_len), q_start=None, kv_len=None, max_q_len=1,
                          all_decode=True, positions=None, token_entry=None)
    cache = SimpleNamespace(group=0, page_size=16, keys=None, values=None)
    part = SimpleNamespace(shares_kv=False, attention_pages=pages, scale=1.0)
    q = torch.zeros(1, 4, 64)
    assert GroupedQueryAttention._attend_chosen(part, q, ctx, cache, None, None) is q
    assert asked == [want]


@pytest.mark.parametrize("head_dim,taken", [(16, True), (128, True), (256, True), (8, False), (24, False), (272, False)])
def test_head_sizes_are_refused_when_a_model_is_loaded(head_dim, taken):
    from types import SimpleNamespace

    from llm_runtime_study_b200.cache.manager import CacheLayout
    from llm_runtime_study_b200.engine.runtime import _check_attention_pages
    from llm_runtime_study_b200.errors import EngineError
    from llm_runtime_study_b200.parts.base import PagedKV

    needs = [PagedKV(2, 64, window=9), PagedKV(2, head_dim, page_tensors=(("bounds", (2, 2, head_dim)),))]
    model = SimpleNamespace(cache_layout=lambda: CacheLayout.from_requirements(needs))
    loaded = SimpleNamespace(model=model, runtime=SimpleNamespace(attention_pages=8))
    if taken:
        assert _check_attention_pages(loaded) is loaded
    else:
        with pytest.raises(EngineError, match="head sizes"):
            _check_attention_pages(loaded)


def test_no_static_is_shared_by_libraries_that_configure_kernels_of_their_own():
    """What a library remembers of its kernels' configuration must not be one object for all builds of the same source (exported names of
    the libraries that are built)."""

    import collections
    import shutil
    import subprocess

    from llm_runtime_study_b200.csrc import build

    for head_dim in range(16, 257, 16):
        sparse_pages.library_name(head_dim)
    specs = native.library_specs()
    paths = [build.library_path(name, sources, native.library_defines(name))[0] for name, sources in specs.items()]
    built = [path for path in paths if path.is_file()]
    if not built or shutil.which("nm") is None:
        pytest.skip("no libraries are built here")
    shared = collections.Counter()
    for path in built:
        names = subprocess.run(["nm", "-D", "--defined-only", str(path)], capture_output=True, text=True, check=True).stdout.splitlines()
        shared.update(name.split()[-1] for name in names if name.split()[-2] == "u")
    assert [name for name, n in shared.items() if n > 1 and name.endswith("4once")] == []


def test_tables_are_current_when_nothing_of_them_changed():
    """``DeviceTables.current`` says of random histories (pages taken, given back by a window, slots reused) what ``changes`` says."""

    import random
    from types import SimpleNamespace

    from llm_runtime_study_b200.cache.tables import DeviceTables

    rng = random.Random(3)
    tables = DeviceTables(4, [20, 20], torch.device("cpu"))
    copies = [t.tolist() for t in tables.tensors]
    live, seen = {}, {True: 0, False: 0}
    for step in range(3000):
        slot = rng.randrange(4)
        if slot not in live or rng.random() < 0.1:
            live[slot] = SimpleNamespace(slot=slot, id=step, tables=[[], []])
        request = live[slot]
        for table in request.tables:
            if len(table) < 20 and rng.random() < 0.2:
                table.extend(rng.randrange(100) for _ in range(rng.randint(1, 3)) if len(table) < 18)
            back = sum(page < 0 for page in table)
            if back < len(table) and rng.random() < 0.1:
                table[back] = -1
        batch = rng.sample(sorted(live), rng.randint(1, len(live)))
        batch = [live[s] for s in batch]
        changes = tables.changes(batch)
        current = tables.current(batch)
        assert current or any(cells.size for cells in changes) or any(not any(r.tables) for r in batch)
        assert not current or not any(cells.size for cells in changes)
        seen[current] += 1
        for g, copy in enumerate(copies):
            for r, c, page in zip(*(cells.tolist() for cells in changes[3 * g : 3 * g + 3])):
                copy[r][c] = page
        tables.sent(batch)
        assert tables.current(batch) and not any(cells.size for cells in tables.changes(batch))
        for request in batch:
            for copy, table in zip(copies, request.tables):
                assert copy[request.slot][: len(table)] == table
    assert min(seen.values()) > 100


@pytest.mark.parametrize("width", [None, 4])
def test_a_block_table_that_is_none_is_refused(host, monkeypatch, width):
    real = page_tables.pointer

    def pointer(t, name, *args, **kwargs):
        if not isinstance(t, torch.Tensor):
            raise KernelError(name)
        return real(t, name, *args, **kwargs)

    monkeypatch.setattr(page_tables, "pointer", pointer)
    with pytest.raises(KernelError, match="block_table"):
        page_tables.step_maps(ints(3, 4), slots=ints(2), kv_len=ints(2), counts=ints(2), page_size=8, num_tokens=4, width=width,
                              out=page_tables.StepMaps(None))
    assert host == []
