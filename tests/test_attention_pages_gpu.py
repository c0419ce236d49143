"""The engine with ``attention_pages``: every token reads a bounded number of pages; and the block tables kept on the device."""

import random

import pytest
import torch

from tests import helpers
from tests.plain import qwen3_plain

pytestmark = pytest.mark.gpu

FIRST, LAST = 1, 2


def chosen_attention(page, budget):
    """``causal_attention`` of the plain model in which every query reads its own choice of pages."""

    def attention(q, k, v, scale, window=None):
        T, nq, d = q.shape
        nkv = k.shape[1]
        group = nq // nkv
        out = torch.empty_like(q)
        for g in range(nkv):
            full = T // page
            low = k[: full * page, g].view(full, page, d).amin(1)
            high = k[: full * page, g].view(full, page, d).amax(1)
            for p in range(T):
                x = q[p, g * group : (g + 1) * group]
                seen = p // page + 1
                pages = list(range(seen))
                if seen > budget:
                    middle = range(FIRST, seen - LAST)
                    score = {c: float(torch.maximum(x * low[c], x * high[c]).sum()) for c in middle}
                    pages = [*range(FIRST), *sorted(middle, key=lambda c: (-score[c], c))[: budget - FIRST - LAST], *range(seen - LAST, seen)]
                keys = [t for c in pages for t in range(c * page, min((c + 1) * page, p + 1))]
                out[p, g * group : (g + 1) * group] = torch.softmax(x @ k[keys, g].T * scale, -1) @ v[keys, g]
        return out

    return attention


def _load(tmp_path, name, dtype, pages):
    from llm_runtime_study_b200.engine.runtime import load

    raw, seed, page = helpers.TINY[name]
    path, weights = helpers.make_model_dir(tmp_path / "m", raw, seed, torch_dtype=dtype)
    return load(path, device="cuda:0", dtype=dtype, attention_pages=pages), raw, weights, page


def _step_all(loaded, page, tokens, cuts, *, max_seq_len=256):
    """Logits of every token of a sequence that is fed in portions."""

    from llm_runtime_study_b200.engine.step import StepEntry

    runner = loaded.make_runner(max_tokens=max_seq_len, page_size=page, max_requests=1, max_seq_len=max_seq_len)
    request, logits, at = runner.manager.admit(), [], 0
    for n in cuts:
        logits.append(runner.step([StepEntry(request, tokens[at : at + n], list(range(n)))]).clone())
        at += n
    return torch.cat(logits), runner, request


@pytest.mark.parametrize("name,budget", [("A", 3), ("A", 7), ("B", 5), ("C", 4)])
def test_logits_match_a_plain_model_that_chooses_pages(tmp_path, monkeypatch, name, budget):
    loaded, raw, weights, page = _load(tmp_path, name, "float32", budget)
    tokens = helpers.random_tokens(random.Random(4), raw["vocab_size"], 15 * page + 3)
    dense = helpers.plain_logits(weights, raw, tokens)
    monkeypatch.setattr(qwen3_plain, "causal_attention", chosen_attention(page, budget))
    want = helpers.plain_logits(weights, raw, tokens)
    assert float((dense - want)[budget * page :].abs().max()) > 1e-3      # the choice matters
    got, _, _ = _step_all(loaded, page, tokens, [len(tokens)])
    torch.testing.assert_close(got.cpu().double(), want, atol=2e-4, rtol=0)
    assert float((got.cpu().double() - dense)[: budget * page].abs().max()) < 2e-4      # nothing to choose from yet


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_budget_of_all_pages_is_attention_over_all_tokens(tmp_path, dtype):
    from llm_runtime_study_b200.engine.runtime import load

    loaded, raw, weights, page = _load(tmp_path, "B", dtype, 64)
    whole = load(tmp_path / "m", device="cuda:0", dtype=dtype)
    tokens = helpers.random_tokens(random.Random(5), raw["vocab_size"], 150)
    for cuts in ([150], [100, 47, 1, 1, 1]):
        a, b = (_step_all(x, page, tokens, cuts)[0] for x in (loaded, whole))
        scale = float(b.float().pow(2).mean().sqrt())
        assert float((a - b).abs().max()) < (1e-4 if dtype == "float32" else 6e-2) * scale


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_budget_beyond_any_sequence_is_one_of_all_pages(tmp_path, dtype):
    """Lists are no longer than the longest sequence's pages, whatever number was given."""

    from llm_runtime_study_b200.engine.runtime import load

    loaded, raw, weights, page = _load(tmp_path, "B", dtype, 10 ** 9)
    fits = load(tmp_path / "m", device="cuda:0", dtype=dtype, attention_pages=-(-256 // page))
    tokens = helpers.random_tokens(random.Random(5), raw["vocab_size"], 150)
    for cuts in ([150], [100, 47, 1, 1, 1]):
        a, b = (_step_all(x, page, tokens, cuts)[0] for x in (loaded, fits))
        assert torch.equal(a, b)


def test_portions_batches_and_new_pages_do_not_change_a_bit(tmp_path):
    """float32: a sequence's logits however its prompt is cut, beside other requests, and after a roll-back."""

    from llm_runtime_study_b200.engine.step import StepEntry

    loaded, raw, _, page = _load(tmp_path, "A", "float32", 4)
    rng = random.Random(6)
    tokens, other = (helpers.random_tokens(rng, raw["vocab_size"], n) for n in (90, 140))
    want, runner, request = _step_all(loaded, page, tokens, [90])
    for cuts in ([1] * 90, [33, 1, 1, 40, 15], [4] * 20 + [10]):
        assert torch.equal(_step_all(loaded, page, tokens, cuts)[0], want)
    # taken back into the middle of a full page, then other tokens, then the same again
    runner.manager.rollback(request, 61)
    runner.step([StepEntry(request, other[:29], [])])
    runner.manager.rollback(request, 61)
    again = runner.step([StepEntry(request, tokens[61:], list(range(29)))])
    assert torch.equal(again, want[61:])
    # beside another request, whose pages lie between this one's
    runner = loaded.make_runner(max_tokens=512, page_size=page, max_requests=2, max_seq_len=256)
    a, b = runner.manager.admit(), runner.manager.admit()
    at, logits = 0, []
    for n in (1, 30, 1, 1, 22, 35):
        out = runner.step([StepEntry(b, other[at : at + n], [0]), StepEntry(a, tokens[at : at + n], list(range(n)))])
        logits.append(out[1:].clone())
        at += n
    assert torch.equal(torch.cat(logits), want)


@pytest.mark.parametrize("least", [0, 10 ** 6])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_captured_decode_equals_eager(tmp_path, monkeypatch, dtype, least):
    from tests.test_generate_gpu import _decode_both_ways
    from llm_runtime_study_b200.engine import step
    from llm_runtime_study_b200.sampling import SamplingConfig

    monkeypatch.setattr(step, "DEVICE_TABLES_MIN_PAGES", least)      # eager steps with tables made on the device, or by the host
    loaded, raw, _, page = _load(tmp_path, "B", dtype, 3)
    rng = random.Random(6)
    prompts = [helpers.random_tokens(rng, raw["vocab_size"], n) for n in (3, 70, 9, 41)]
    live = [[0, 1, 2, 3]] * 12 + [[0, 1, 2]] * 3 + [[0, 1]] * 3
    (eager_ids, eager_logits), (graph_ids, graph_logits) = _decode_both_ways(
        loaded, prompts, live, page=page, max_seq_len=128, sampling=SamplingConfig(temperature=0.8, seed=9))
    assert eager_ids == graph_ids
    for a, b in zip(eager_logits, graph_logits):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_with_preemption_and_reuse(tmp_path, dtype):
    """Through the entry point: a cache too small for all requests at once, so that some are computed anew; float32 gives the same
    tokens as each prompt alone."""

    from llm_runtime_study_b200.engine.engine import Engine

    raw, seed, page = helpers.TINY["A"]
    path, _ = helpers.make_model_dir(tmp_path / "m", raw, seed, torch_dtype=dtype)
    rng = random.Random(8)
    prompts = [helpers.random_tokens(rng, raw["vocab_size"], n) for n in (37, 5, 60, 21, 44)]
    options = dict(device="cuda:0", dtype=dtype, max_seq_len=128, page_size=page, max_tokens_per_step=16, attention_pages=5)

    def tokens(engine, prompts):
        out = {}
        for index, event in engine.generate(prompts, max_new_tokens=24):
            out.setdefault(index, []).append(event.token_id)
        assert engine.cache_manager.all_free
        return out

    engine = Engine.from_model_dir(path, max_batch_size=3, max_cache_tokens=148, **options)
    assert engine.attention_pages == 5
    got = tokens(engine, prompts)
    assert tokens(engine, prompts) == got              # the pages and slots used before
    if dtype == "float32":
        alone = Engine.from_model_dir(path, max_batch_size=1, use_cuda_graph=False, device_sampling=False, **options)
        for i, prompt in enumerate(prompts):
            assert tokens(alone, [prompt])[0] == got[i]
    engine.to(dtype="bfloat16" if dtype == "float32" else "float32")
    assert engine.attention_pages == 5


def test_what_the_engine_refuses(tmp_path):
    from llm_runtime_study_b200.engine.engine import Engine
    from llm_runtime_study_b200.errors import EngineError

    raw, seed, page = helpers.TINY["A"]
    path, _ = helpers.make_model_dir(tmp_path / "m", raw, seed)
    for value in (0, 2, -1, True, 4.0, "8"):
        with pytest.raises(EngineError, match="attention_pages"):
            Engine.from_model_dir(path, device="cuda:0", attention_pages=value)
    with pytest.raises(EngineError, match="no layer"):
        Engine.from_random_weights(helpers.SORULIX_A, device="cuda:0", dtype="float32", max_seq_len=32, attention_pages=8)


def test_the_command_line_takes_the_option(tmp_path):
    import io

    from llm_runtime_study_b200.cli import main

    raw, seed, page = helpers.TINY["A"]
    path, weights = helpers.make_model_dir(tmp_path / "m", raw, seed)
    prompt = " ".join(str(t) for t in helpers.random_tokens(random.Random(1), raw["vocab_size"], 70))
    texts = []
    for pages in ("3", "64"):
        out, err = io.StringIO(), io.StringIO()
        options = ["--model", str(path), "--prompt-ids", prompt, "--max-new-tokens", "12", "--dtype", "float32", "--page-size", str(page),
                   "--max-seq-len", "128", "--no-metrics"]
        assert main([*options, "--attention-pages", pages], output=out, error=err) == 0, err.getvalue()
        texts.append(out.getvalue())
        assert main([*options, "--attention-pages", "2"], output=out, error=err) == 2 and "attention_pages" in err.getvalue()
    out = io.StringIO()
    assert main(options, output=out, error=io.StringIO()) == 0
    assert texts[1] == out.getvalue() and texts[0].split()       # a budget of all pages reads them all


def test_the_cache_counts_what_it_keeps_per_page():
    from llm_runtime_study_b200.cache.manager import CacheLayout, CacheManager
    from llm_runtime_study_b200.parts.base import PagedKV

    plain, kept = (CacheManager(CacheLayout.from_requirements([PagedKV(2, 16, page_tensors=t)] * 3), max_tokens=64, page_size=8, max_requests=2,
                                dtype=torch.bfloat16, device="cuda") for t in ((), (("bounds", (2, 2, 16)),)))
    assert kept.groups[0].tensors["bounds"].shape == (3, 8, 2, 2, 16) and kept.layer_cache(1).tensors["bounds"].shape == (8, 2, 2, 16)
    assert kept.num_bytes - plain.num_bytes == 3 * 8 * 64 * 2
    assert kept.bytes_per_token() - plain.bytes_per_token() == 3 * 8 * 2


# ------------------------------------------------------------------------------------------------ tables on the device
class _Nothing:
    """A model of no layers, for the runner's bookkeeping."""

    def bind_cache(self, manager):
        pass

    def forward(self, ctx):
        return None


@pytest.mark.parametrize("least", [0, 40, 10 ** 6])
@pytest.mark.parametrize("seed", range(3))
def test_tables_on_the_device_follow_the_host_s(monkeypatch, seed, least):
    """(``least``: pages from which a step's tables are made on the device; all of them, some, none.)  Random steps over three groups of pages (a window, a page size of its own): admission, portions, decoding, roll-backs,
    release and reuse of slots; block tables, positions and slot maps equal what the host's tables say."""

    from llm_runtime_study_b200.cache.manager import CacheLayout, CacheManager
    from llm_runtime_study_b200.engine.step import StepEntry, StepRunner
    from llm_runtime_study_b200.engine import step
    from llm_runtime_study_b200.parts.base import PagedKV, Runtime

    monkeypatch.setattr(step, "DEVICE_TABLES_MIN_PAGES", least)
    rng = random.Random(seed)
    layout = CacheLayout.from_requirements([PagedKV(1, 16), PagedKV(1, 16, window=9), PagedKV(1, 16, page_size=5)])
    device = torch.device("cuda:0")
    manager = CacheManager(layout, max_tokens=520, page_size=4, max_requests=5, dtype=torch.float32, device=device, max_seq_len=90)
    runner = StepRunner(_Nothing(), manager, Runtime(device, torch.float32), vocab_size=50, max_positions=90)
    live = []
    for _ in range(120):
        if live and rng.random() < 0.15:
            manager.release(live.pop(rng.randrange(len(live))))
        while manager.free_slots and rng.random() < 0.5:
            live.append(manager.admit())
        batch = [r for r in rng.sample(live, len(live)) if r.length < 80][: rng.randint(1, 5)]
        if not batch:
            continue
        for r in batch:
            if r.length > 20 and rng.random() < 0.1 and all(t[-1] >= 0 for t in r.tables):
                manager.rollback(r, r.length - rng.randint(0, 3))
        decode = rng.random() < 0.5
        entries = [StepEntry(r, [1] * (1 if decode else rng.randint(1, min(20, 90 - r.length)))) for r in batch]
        ctx = runner.build_context(entries)
        at = 0
        assert ctx.q_start.tolist() == [sum(ctx.q_lens[:i]) for i in range(len(batch) + 1)]
        for i, (entry, n, length) in enumerate(zip(entries, ctx.q_lens, ctx.kv_lens)):
            assert ctx.positions[at : at + n].tolist() == list(range(length - n, length))
            assert ctx.token_entry[at : at + n].tolist() == [i] * n
            for g, pool in enumerate(manager.groups):
                table = entry.request.tables[g]
                held = table[: -(-length // pool.page_size)]
                row = ctx.block_table(g)[i].tolist()
                # behind its last page a row ends; one put together by the host shows pages taken in advance, too
                rest = [-1] * (len(row) - len(held)) if least == 0 else (table[len(held) :] + [-1] * len(row))[: len(row) - len(held)]
                assert row[: len(held)] == held and (row[len(held) :] == rest or set(row[len(held) :]) <= {-1}), (g, i)
                want = [table[p // pool.page_size] * pool.page_size + p % pool.page_size for p in range(length - n, length)]
                assert ctx.slot_map(g)[at : at + n].tolist() == want
            at += n
        for entry, length in zip(entries, ctx.kv_lens):
            manager.commit(entry.request, length)
        manager.check()


@pytest.mark.parametrize("width", [8, 6])
def test_slot_load_and_the_block_table_in_one_launch(width):
    from llm_runtime_study_b200.cache.slots import SLOT_WORDS, SlotRecord
    from llm_runtime_study_b200.errors import KernelError
    from llm_runtime_study_b200.ops import page_tables, slots as slot_ops

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    records = torch.zeros((6, SLOT_WORDS), dtype=torch.int32)
    records[1] = torch.tensor(SlotRecord(position=0, last_token=7).words(), dtype=torch.int32)
    records[3] = torch.tensor(SlotRecord(position=15, last_token=-1).words(), dtype=torch.int32)
    records[4] = torch.tensor(SlotRecord(position=16, last_token=9).words(), dtype=torch.int32)
    tables = torch.arange(6 * width, dtype=torch.int32).view(6, width).cuda()
    slots = ints([4, 5, 1, 3])
    got, want = [[records.cuda(), *(torch.full((4,), 77, dtype=torch.int32, device="cuda") for _ in range(3))] for _ in range(2)]
    block = torch.full((5, width), 77, dtype=torch.int32, device="cuda")
    page_tables.slot_load_maps(got[0], slots, *got[1:], tables=tables, page_size=4, block_table=block)
    slot_ops.slot_load(want[0], slots, *want[1:])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    rows = tables.tolist()
    assert block[:4].tolist() == [rows[4][:5] + [-1] * (width - 5), [-1] * width, rows[1][:1] + [-1] * (width - 1),
                                  rows[3][:4] + [-1] * (width - 4)]
    assert bool((block[4] == 77).all())
    for bad in (dict(block_table=block[:3]), dict(page_size=0), dict(tables=tables[:, :3])):
        with pytest.raises(KernelError):
            page_tables.slot_load_maps(got[0], slots, *got[1:], **(dict(tables=tables, page_size=4, block_table=block) | bad))
