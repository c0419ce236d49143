"""Timed cases of attention over chosen pages of a long cache, and of the page maps that such steps need.

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare(case, seed)`` makes what a serving
program holds before the call, ``run(state)`` is one pass through an operator, ``work(case)`` says what the pass cannot do
without, ``exact(case, seed)`` computes the same outputs in 64 bits.

Kinds of cases (``case["op"]``):

* ``maps``: the pages that requests have taken go into the table on the device, and a step's block tables, positions and slot
  maps are built there from the requests' lengths (``page_table_set``, ``step_maps``).
* ``bounds``: for the pages that became full in a step, the least and the greatest value of every key channel
  (``page_bounds``).
* ``choose``: every query row scores the pages it sees by their bounds and keeps the best (``choose_pages``): the score of a
  page is the sum over the group's query heads and the channels of ``max(q * low, q * high)``, the first page and the last
  two are always kept, equal scores go to the lower page.
* ``attend``: softmax attention of every query row over the pages chosen for it (``paged_attention_chosen``).
* ``layer``: the three in a row, as an attention layer issues them.

Sizes: ``requests`` sequences of about ``context`` tokens (``ragged``: of falling length), ``tokens`` of them new in this step
(1: decoding; more: a prompt portion), ``heads`` query heads over ``kv_heads`` key and value heads of ``head_dim``, pages of
``page`` tokens, at most ``budget`` pages a query row.
"""

from __future__ import annotations

import math
import random

import torch

own = False

FIRST, LAST = 1, 2          # pages at the start and at the end of what a row sees that it always reads
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------- cases
def _case(op, requests, context, tokens, page, budget=0, heads=32, kv_heads=8, head_dim=128, dtype="bfloat16", ragged=True):
    return {"op": op, "requests": requests, "context": context, "tokens": tokens, "page": page, "budget": budget, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "ragged": ragged}


def listed() -> list[dict]:
    cases = {
        # one decode step of a full batch of long requests: every row of the block table anew
        "maps_decode_64": _case("maps", 64, 32768, 1, 16),
        # a step of prompt portions: thousands of tokens' positions and slots
        "maps_prompt": _case("maps", 7, 65536, 1200, 32),
        # the pages a step of prompt portions fills, 32 query / 8 key heads of 128
        "bounds_prompt": _case("bounds", 5, 8192, 2048, 16),
        # the smallest call: one float32 request whose last page becomes full, small heads
        "bounds_one_f32": _case("bounds", 1, 640, 1, 16, heads=8, kv_heads=2, head_dim=64, dtype="float32", ragged=False),
        # one request far into a long document, decoding
        "choose_one": _case("choose", 1, 32768, 1, 16, 128, ragged=False),
        # a batch of long requests of different lengths, 40 query heads over 8
        "choose_batch": _case("choose", 32, 65521, 1, 32, 64, heads=40),
        # prompt portions behind what is cached: every token chooses for itself
        "choose_prompt": _case("choose", 2, 16384, 500, 16, 128, heads=16),
        "attend_one": _case("attend", 1, 32768, 1, 16, 128, ragged=False),
        # 64 query heads over 8, large pages, a full batch
        "attend_batch": _case("attend", 64, 16384, 1, 64, 32, heads=64),
        "attend_prompt": _case("attend", 2, 16384, 500, 16, 128, heads=16),
        # what one attention layer runs in a decode step of a batch
        "layer_decode": _case("layer", 16, 32760, 1, 16, 128),
        # the float32 path: short portions of prompts, head size 64
        "layer_f32": _case("layer", 3, 4099, 37, 16, 24, heads=8, kv_heads=2, head_dim=64, dtype="float32"),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["maps", "bounds", "choose", "choose", "attend", "attend", "layer", "layer"])
    page = rng.choice([16, 16, 32, 64])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    head_dim = rng.choice([64, 128, 128])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    budget = _log(rng, 4, 128)
    if rng.random() < 0.65 or op == "maps" and rng.random() < 0.5:      # decoding
        requests, tokens = _log(rng, 1, 48), 1
        context = _log(rng, 1, min(60000, 500000 // requests))
    else:                                                               # prompt portions
        requests = _log(rng, 1, 6)
        tokens = _log(rng, 2, (4000 if op in ("maps", "bounds") else 700) // requests)
        context = tokens + _log(rng, 1, 12000)
        budget = min(budget, 64)
    if op in ("maps", "choose"):        # sequences of more pages than there are choices
        context = max(context, tokens + 40 * page)
        budget = min(budget, context // (2 * page))
    if op == "bounds":                  # the first request's last page becomes full
        context = -(-context // page) * page
    return _case(op, requests, context, tokens, page, budget, kv_heads * group, kv_heads, head_dim, dtype, rng.random() < 0.7)


def _counts(case: dict) -> list[int]:
    """New tokens of every request."""

    n, tokens = case["requests"], case["tokens"]
    if tokens == 1 or not case["ragged"]:
        return [tokens] * n
    return [max(1, tokens - (tokens * r) // (2 * n) - r) for r in range(n)]


def _lengths(case: dict) -> list[int]:
    """Every request's length once the step has run."""

    n, context = case["requests"], case["context"]
    if not case["ragged"]:
        return [context] * n
    return [max(count, context - (3 * context * r) // (4 * n) - 5 * r) for r, count in enumerate(_counts(case))]


def _pages(case: dict) -> list[int]:
    return [-(-length // case["page"]) for length in _lengths(case)]


def _width(case: dict) -> int:
    return -(-max(_pages(case)) // 4) * 4


def _full(case: dict) -> int:
    """Pages that become full in the step."""

    return sum(length // case["page"] - (length - count) // case["page"] for length, count in zip(_lengths(case), _counts(case)))


def work(case: dict) -> dict:
    counts, lengths, pages = _counts(case), _lengths(case), _pages(case)
    size = 4 if case["dtype"] == "float32" else 2
    page, d, heads, kv_heads = case["page"], case["head_dim"], case["heads"], case["kv_heads"]
    tokens = sum(counts)
    moved = flops = 0
    if case["op"] == "maps":
        moved = 4 * sum(pages) + 4 * case["requests"] * _width(case) + 16 * tokens + 16 * case["requests"]
        flops = 2 * tokens
    if case["op"] in ("bounds", "layer"):
        moved += _full(case) * kv_heads * d * size * (page + 2)
        flops += 2 * _full(case) * kv_heads * d * page
    if case["op"] in ("choose", "layer"):
        moved += sum(pages) * (kv_heads * 2 * d * size + 4) + tokens * heads * d * size + tokens * kv_heads * case["budget"] * 4
        flops += 4 * d * kv_heads * sum((length - i) // page for length, count in zip(lengths, counts) for i in range(count))
    if case["op"] in ("attend", "layer"):
        for length, count, held in zip(lengths, counts, pages):
            keys = min(length, case["budget"] * page)
            moved += keys * kv_heads * 2 * d * size             # the pages of one row at least
            moved += count * heads * d * size * 2 + (count * kv_heads * case["budget"] * 4 if case["op"] == "attend" else 0)
            flops += 4 * d * heads * count * keys
    return {"bytes": moved, "flops": max(flops, 1)}


# --------------------------------------------------------------------------------------------------------------- inputs
def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, page, d = DTYPES[case["dtype"]], case["page"], case["head_dim"]
    counts, lengths, pages, width = _counts(case), _lengths(case), _pages(case), _width(case)
    n, total, tokens = case["requests"], sum(pages), sum(counts)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    for r, at in enumerate(_starts(pages)):
        table[r, : pages[r]] = order[at : at + pages[r]]
    state = {"case": case, "counts": counts, "lengths": lengths, "pages": pages, "width": width, "tokens": tokens}
    kv_len, new = ints(lengths), ints(counts)
    if case["op"] == "maps":
        # the table of all request slots: rows in another order than the step's, the new pages not in it yet
        slots = torch.randperm(n + 3, generator=g, device="cuda")[:n]
        tables = torch.full((n + 3, width), -1, dtype=torch.int32, device="cuda")
        tables[slots] = table
        before = [-(-(length - count) // page) for length, count in zip(lengths, counts)]
        row = torch.cat([slots[r].expand(pages[r] - before[r]) for r in range(n)])
        column = torch.cat([torch.arange(before[r], pages[r], device="cuda") for r in range(n)])
        state.update(tables=tables, slots=slots.to(torch.int32), kv_len=kv_len, new=new, rows=row.to(torch.int32),
                     columns=column.to(torch.int32), taken=tables[row, column].clone())
        tables[row, column] = -1
        return state
    entry = torch.repeat_interleave(torch.arange(n, device="cuda"), new.long(), output_size=tokens)
    q_start = ints(_starts(counts) + [tokens])
    state.update(table=table, kv_len=kv_len, q_start=q_start, entry=entry.to(torch.int32),
                 positions=torch.cat([torch.arange(length - count, length, device="cuda") for length, count in zip(lengths, counts)]).to(torch.int32))
    if case["op"] != "bounds":
        # queries and keys as a norm per head leaves them: numbers of size one in every channel
        state["q"] = torch.randn((tokens, case["heads"], d), generator=g, device="cuda").to(dtype)
    if case["op"] != "choose":
        state["keys"], state["values"] = (_rows(g, total, case, dtype) for _ in range(2))
    if case["op"] == "choose":
        centre = torch.randn((total, case["kv_heads"], d), generator=g, device="cuda") * 0.7
        spread = torch.rand((2, total, case["kv_heads"], d), generator=g, device="cuda") + 0.5
        state["bounds"] = torch.stack((centre - spread[0], centre + spread[1]), dim=2).to(dtype).contiguous()
    if case["op"] in ("bounds", "layer"):
        state["bounds"] = torch.stack((state["keys"].amin(dim=2), state["keys"].amax(dim=2)), dim=2).contiguous()
    if case["op"] == "attend":
        state["chosen"] = _any_pages(g, state)
    return state


def _starts(sizes: list[int]) -> list[int]:
    out, at = [], 0
    for size in sizes:
        out.append(at)
        at += size
    return out


def _rows(g, total: int, case: dict, dtype) -> torch.Tensor:
    """Rows of the pool ``[pages, kv heads, page, head_dim]``; those of a page are alike, as those of a passage are."""

    shape = (total, case["kv_heads"], case["page"], case["head_dim"])
    rows = torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(0.7)
    return rows.add_(torch.randn((total, case["kv_heads"], 1, case["head_dim"]), generator=g, device="cuda", dtype=dtype), alpha=0.7)


def _any_pages(g, state: dict) -> torch.Tensor:
    """Pages for every row and kv head: its last two, the first and others at random, ascending, -1 behind."""

    case = state["case"]
    n, k, width = state["tokens"], case["budget"], state["width"]
    out = torch.full((n, case["kv_heads"], k), -1, dtype=torch.int32, device="cuda")
    column = torch.arange(width, device="cuda")
    for at in range(0, n, 256):
        seen = (state["positions"][at : at + 256].long() // case["page"] + 1)[:, None, None]
        rank = torch.rand((seen.shape[0], case["kv_heads"], width), generator=g, device="cuda")
        rank = torch.where((column < FIRST) | (column >= seen - LAST), 2.0, rank)
        rank = torch.where(column >= seen, -1.0, rank)
        best = rank.topk(min(k, width), dim=-1)
        pages = torch.where(best.values >= 0, best.indices, width).sort(dim=-1).values
        out[at : at + 256, :, : pages.shape[-1]] = torch.where(pages < width, pages, -1).to(torch.int32)
    return out


# ------------------------------------------------------------------------------------------------------------------ run
def run(state: dict):
    case = state["case"]
    if own:
        return _run_own(state)
    if case["op"] == "maps":
        return _plain_maps(state)
    if case["op"] == "bounds":
        return _plain_bounds(state)
    if case["op"] == "choose":
        return _plain_choose(state)
    if case["op"] == "attend":
        return _plain_attend(state, state["chosen"])
    bounds = _plain_bounds(state)
    chosen = _plain_choose(state)
    return {"bounds": bounds, "chosen": chosen, "out": _plain_attend(state, chosen)}


def _run_own(s: dict):
    from llm_runtime_study_b200.ops import page_tables, sparse_pages

    case = s["case"]
    if case["op"] == "maps":
        page_tables.page_table_set(s["tables"], rows=s["rows"], columns=s["columns"], pages=s["taken"])
        maps = page_tables.step_maps(s["tables"], slots=s["slots"], kv_len=s["kv_len"], counts=s["new"], page_size=case["page"],
                                     num_tokens=s["tokens"])
        return {"tables": s["tables"], "block_table": maps.block_table, "q_start": maps.q_start, "positions": maps.positions,
                "token_entry": maps.token_entry, "slot_map": maps.slot_map}
    scale = case["head_dim"] ** -0.5
    rows = {"positions": s["positions"], "token_entry": s["entry"], "block_table": s["table"]}

    def bounds():
        sparse_pages.page_bounds(s["keys"], s["bounds"], block_table=s["table"], q_start=s["q_start"], kv_len=s["kv_len"],
                                 max_q_len=max(s["counts"]))
        return s["bounds"]

    def choose():
        return sparse_pages.choose_pages(s["q"], s["bounds"], page_size=case["page"], budget=case["budget"], first=FIRST, last=LAST,
                                         **rows)

    def attend(chosen):
        return sparse_pages.paged_attention_chosen(s["q"], s["keys"], s["values"], chosen, scale=scale, **rows)

    if case["op"] == "bounds":
        return bounds()
    if case["op"] == "choose":
        return choose()
    if case["op"] == "attend":
        return attend(s["chosen"])
    bounds()
    chosen = choose()
    return {"bounds": s["bounds"], "chosen": chosen, "out": attend(chosen)}


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_maps(s: dict) -> dict:
    case, tables, n = s["case"], s["tables"], s["case"]["requests"]
    page = case["page"]
    tables[s["rows"].long(), s["columns"].long()] = s["taken"]
    q_start = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    q_start[1:] = torch.cumsum(s["new"], 0)
    entry = torch.repeat_interleave(torch.arange(n, device="cuda"), s["new"].long(), output_size=s["tokens"])
    start = (s["kv_len"] - s["new"]).clamp(min=0)
    positions = start[entry] + torch.arange(s["tokens"], device="cuda") - q_start[entry]
    held = (s["kv_len"] + page - 1) // page
    table = torch.where(torch.arange(s["width"], device="cuda") < held[:, None], tables[s["slots"].long()], -1)
    of = table[entry, positions // page].long()
    slot = torch.where(of >= 0, of * page + positions % page, -1)
    return {"tables": tables, "block_table": table, "q_start": q_start, "positions": positions.to(torch.int32),
            "token_entry": entry.to(torch.int32), "slot_map": slot}


def _plain_bounds(s: dict) -> torch.Tensor:
    page, bounds = s["case"]["page"], s["bounds"]
    column = torch.arange(s["width"], device="cuda")
    new = s["q_start"][1:] - s["q_start"][:-1]
    full = (column >= ((s["kv_len"] - new) // page)[:, None]) & (column < (s["kv_len"] // page)[:, None])
    ids = s["table"][full].long()
    for at in range(0, ids.numel(), 4096):
        part = ids[at : at + 4096]
        keys = s["keys"][part].float()
        bounds[part] = torch.stack((keys.amin(dim=2), keys.amax(dim=2)), dim=2).to(bounds.dtype)
    return bounds


def _plain_choose(s: dict) -> torch.Tensor:
    case, q = s["case"], s["q"]
    kv_heads, k, page, width = case["kv_heads"], case["budget"], case["page"], s["width"]
    grouped = q.view(q.shape[0], kv_heads, -1, case["head_dim"]).double()
    up, down = grouped.clamp(min=0).sum(2), grouped.clamp(max=0).sum(2)            # [rows, kv heads, d]
    out = torch.full((q.shape[0], kv_heads, k), -1, dtype=torch.int32, device="cuda")
    if max(s["counts"]) == 1:
        parts = [(slice(at, min(at + 16, q.shape[0])), slice(at, min(at + 16, q.shape[0]))) for at in range(0, q.shape[0], 16)]
    else:
        parts = []
        for r, (at, count) in enumerate(zip(_starts(s["counts"]), s["counts"])):
            parts += [(slice(at + i, at + min(i + 128, count)), slice(r, r + 1)) for i in range(0, count, 128)]
    column = torch.arange(width, device="cuda")
    for rows, entries in parts:
        table = s["table"][entries].long()
        b = s["bounds"][table.clamp(min=0)].double()                                 # [entries, width, kv heads, 2, d]
        if b.shape[0] == 1:
            low, high = b[0, :, :, 0].permute(1, 2, 0), b[0, :, :, 1].permute(1, 2, 0)
            score = (up[rows].transpose(0, 1) @ high + down[rows].transpose(0, 1) @ low).transpose(0, 1)
        else:
            low, high = b[:, :, :, 0].permute(0, 2, 3, 1), b[:, :, :, 1].permute(0, 2, 3, 1)
            score = (up[rows][:, :, None] @ high + down[rows][:, :, None] @ low)[:, :, 0]
        score = score.float()                                                        # [rows, kv heads, width]
        seen = (s["positions"][rows].long() // page + 1)[:, None, None]
        kind = torch.where((column < FIRST) | (column >= seen - LAST), 0, 1)
        kind = torch.where((column >= seen) | (table < 0)[:, None], 2, kind).expand_as(score)
        best = score.argsort(dim=-1, descending=True, stable=True)                   # lower pages first among equals
        kept = kind.gather(-1, best)
        best = best.gather(-1, kept.argsort(dim=-1, stable=True))[..., :k]
        best = torch.where(kind.gather(-1, best) < 2, best, width).sort(dim=-1).values
        out[rows, :, : best.shape[-1]] = torch.where(best < width, best, -1).to(torch.int32)
    return out


def _plain_attend(s: dict, chosen: torch.Tensor) -> torch.Tensor:
    case, q = s["case"], s["q"]
    kv_heads, d, page, k = case["kv_heads"], case["head_dim"], case["page"], case["budget"]
    out = torch.empty_like(q)
    step = max(1, (1 << 28) // (kv_heads * k * page * d * 4))
    head = torch.arange(kv_heads, device="cuda")[:, None]
    offset = torch.arange(page, device="cuda")
    for at in range(0, q.shape[0], step):
        rows = slice(at, at + step)
        c = chosen[rows].long()
        table = s["table"][s["entry"][rows].long()].long()
        ids = table[:, None].expand(-1, kv_heads, -1).gather(-1, c.clamp(min=0))
        at_key = (c * page)[..., None] + offset                                      # [rows, kv heads, k, page]
        hidden = (c < 0)[..., None] | (at_key > s["positions"][rows].long()[:, None, None, None])
        keys = s["keys"][ids, head].float().flatten(2, 3)                            # [rows, kv heads, keys, d]
        values = s["values"][ids, head].float().flatten(2, 3)
        grouped = q[rows].view(keys.shape[0], kv_heads, -1, d).float()
        score = (grouped @ keys.transpose(-1, -2)) * d ** -0.5
        score = score.masked_fill(hidden.flatten(2, 3)[:, :, None], -math.inf)
        weight = torch.exp(score - score.amax(dim=-1, keepdim=True))
        out[rows] = ((weight @ values) / weight.sum(dim=-1, keepdim=True)).reshape(q[rows].shape).to(q.dtype)
    return out


# ------------------------------------------------------------------------------------------------- from the definitions
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "maps":
        return _exact_maps(s)
    if case["op"] == "bounds":
        return _exact_bounds(s)
    if case["op"] == "choose":
        return _exact_choose(s, s["bounds"].double())
    if case["op"] == "attend":
        return _exact_attend(s, s["chosen"])
    bounds = _exact_bounds(s)
    chosen = _exact_choose(s, bounds)
    return {"bounds": bounds, "chosen": chosen, "out": _exact_attend(s, chosen)}


def _exact_maps(s: dict) -> dict:
    page = s["case"]["page"]
    tables = s["tables"].tolist()
    for row, column, of in zip(s["rows"].tolist(), s["columns"].tolist(), s["taken"].tolist()):
        tables[row][column] = of
    block, start, positions, entry, slots = [], [0], [], [], []
    for r, slot in enumerate(s["slots"].tolist()):
        length, count = s["lengths"][r], s["counts"][r]
        block.append([tables[slot][c] if c * page < length else -1 for c in range(s["width"])])
        start.append(start[-1] + count)
        for p in range(length - count, length):
            positions.append(p)
            entry.append(r)
            slots.append(block[r][p // page] * page + p % page)
    made = {"tables": tables, "block_table": block, "q_start": start, "positions": positions, "token_entry": entry}
    made = {name: torch.tensor(value, dtype=torch.int32, device="cuda") for name, value in made.items()}
    return {**made, "slot_map": torch.tensor(slots, dtype=torch.int64, device="cuda")}


def _exact_bounds(s: dict) -> torch.Tensor:
    page, bounds = s["case"]["page"], s["bounds"].double()
    for r, (length, count) in enumerate(zip(s["lengths"], s["counts"])):
        for c in range((length - count) // page, length // page):
            tile = s["keys"][int(s["table"][r, c])].double()
            bounds[int(s["table"][r, c]), :, 0] = tile.min(dim=1).values
            bounds[int(s["table"][r, c]), :, 1] = tile.max(dim=1).values
    return bounds


def _exact_choose(s: dict, bounds: torch.Tensor) -> torch.Tensor:
    """Head by head and sequence by sequence, the score as the sum of greater products."""

    case = s["case"]
    group, k, page = case["heads"] // case["kv_heads"], case["budget"], case["page"]
    out = torch.full((s["tokens"], case["kv_heads"], k), -1, dtype=torch.int32)
    row = 0
    for r, (length, count) in enumerate(zip(s["lengths"], s["counts"])):
        held = bounds[s["table"][r, : -(-length // page)].long()]
        for h in range(case["kv_heads"]):
            low, high = held[:, h, 0].T.contiguous(), held[:, h, 1].T.contiguous()
            for at in range(0, count, 64):
                score = None
                for j in range(h * group, (h + 1) * group):
                    q = s["q"][row + at : row + min(at + 64, count), j].double()
                    part = q.relu() @ high - (-q).relu() @ low                     # max(q low, q high) = q high for q > 0, else q low
                    score = part if score is None else score + part
                for i, line in enumerate(score.float().cpu().tolist()):
                    seen = (length - count + at + i) // page + 1
                    always = [c for c in range(seen) if c < FIRST or c >= seen - LAST]
                    others = sorted((c for c in range(FIRST, seen - LAST)), key=lambda c: (-line[c], c))
                    picked = sorted((always + others)[: max(k, len(always))])
                    out[row + at + i, h, : len(picked)] = torch.tensor(picked, dtype=torch.int32)
        row += count
    return out.cuda()


def _exact_attend(s: dict, chosen: torch.Tensor) -> torch.Tensor:
    case = s["case"]
    group, d, page = case["heads"] // case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lanes = torch.arange(page, device="cuda")
    step = max(1, (1 << 26) // (case["budget"] * page * d))
    for h in range(case["kv_heads"]):
        for at in range(0, s["tokens"], step):
            pages = chosen[at : at + step, h].long()
            entry = s["entry"][at : at + step].long()
            ids = s["table"][entry[:, None], pages.clamp(min=0)].long()
            where = (pages[..., None] * page + lanes).flatten(1)
            seen = (pages >= 0).repeat_interleave(page, dim=1) & (where <= s["positions"][at : at + step, None].long())
            k = s["keys"][ids, h].double().flatten(1, 2)
            v = s["values"][ids, h].double().flatten(1, 2)
            for j in range(h * group, (h + 1) * group):
                logit = (k * s["q"][at : at + step, None, j].double()).sum(-1) / math.sqrt(d)
                p = torch.softmax(logit.masked_fill(~seen, -math.inf), dim=-1)
                out[at : at + step, j] = (p[..., None] * v).sum(1)
    return out
