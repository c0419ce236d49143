"""Plain float64 forms of the page maps, the page bounds, the choice of pages and attention over chosen pages."""

import math

import torch


def step_maps(tables, slots, kv_len, counts, page_size, width):
    """(block table, q_start, positions, token_entry, slot_map) as lists of ints."""

    block, start, positions, entry, slot_map = [], [0], [], [], []
    for r, slot in enumerate(slots):
        held = -(-kv_len[r] // page_size)
        known = 0 <= slot < len(tables)
        row = [tables[slot][c] if known and c < min(held, len(tables[slot])) else -1 for c in range(width)]
        full = [tables[slot][c] if known and c < held else -1 for c in range(len(tables[slot]))] if known else []
        block.append(row)
        start.append(start[-1] + counts[r])
        for i in range(counts[r]):
            p = max(kv_len[r] - counts[r], 0) + i
            column = p // page_size
            page = full[column] if column < len(full) else -1
            positions.append(p)
            entry.append(r)
            slot_map.append(page * page_size + p % page_size if page >= 0 else -1)
    return block, start, positions, entry, slot_map


def page_bounds(keys, bounds, block_table, kv_len, counts):
    """A copy of ``bounds`` with the pages that became full written anew."""

    out, page_size = bounds.clone(), keys.shape[2]
    for r, (length, count) in enumerate(zip(kv_len, counts)):
        for c in range(max(length - count, 0) // page_size, min(length // page_size, block_table.shape[1])):
            page = int(block_table[r, c])
            if 0 <= page < keys.shape[0]:
                out[page, :, 0] = keys[page].amin(dim=1)
                out[page, :, 1] = keys[page].amax(dim=1)
    return out


def choose_pages(q, bounds, positions, token_entry, block_table, page_size, budget, first, last):
    """int32 [n, kv heads, budget], page by page: the sum of max(q low, q high) over heads and channels, the heads'
    positive and negative parts added up first."""

    n, heads, d = q.shape
    kv_heads = bounds.shape[1]
    group = heads // kv_heads
    out = torch.full((n, kv_heads, budget), -1, dtype=torch.int32)
    for i in range(n):
        p, e = int(positions[i]), int(token_entry[i])
        if p < 0 or not 0 <= e < block_table.shape[0]:
            continue
        seen = min(p // page_size + 1, block_table.shape[1])
        for g in range(kv_heads):
            ranked = []
            for c in range(seen):
                page = int(block_table[e, c])
                if not 0 <= page < bounds.shape[0]:
                    continue
                x = q[i, g * group : (g + 1) * group].double()
                score = (x.clamp(max=0).sum(0) * bounds[page, g, 0].double() + x.clamp(min=0).sum(0) * bounds[page, g, 1].double()).sum()
                score = float(score.float())
                always = c < first or c >= seen - last
                ranked.append((0 if always else 1, 0 if math.isnan(score) else 1, 0.0 if math.isnan(score) else -score, c))
            kept = sorted(r[3] for r in sorted(ranked)[:budget])
            out[i, g, : len(kept)] = torch.tensor(kept, dtype=torch.int32)
    return out


def attend_chosen(q, keys, values, chosen, positions, token_entry, block_table, scale):
    """(output, weighted sum of |v|, keys seen at most, most of sum |q k| scale) in float64."""

    n, heads, d = q.shape
    pages, kv_heads, page_size, _ = keys.shape
    group = heads // kv_heads
    out = torch.zeros((n, heads, d), dtype=torch.float64)
    size = torch.zeros_like(out)
    most, spread = 0, 0.0
    for i in range(n):
        p, e = int(positions[i]), int(token_entry[i])
        for g in range(kv_heads):
            ks, vs = [], []
            for c in chosen[i, g].tolist():
                if not (0 <= e < block_table.shape[0] and 0 <= c < block_table.shape[1]):
                    continue
                page = int(block_table[e, c])
                seen = min(page_size, p - c * page_size + 1)
                if 0 <= page < pages and seen > 0:
                    ks.append(keys[page, g, :seen].double())
                    vs.append(values[page, g, :seen].double())
            if not ks:
                continue
            k, v = torch.cat(ks), torch.cat(vs)
            x = q[i, g * group : (g + 1) * group].double()
            w = torch.softmax(x @ k.T * scale, dim=-1)
            out[i, g * group : (g + 1) * group] = w @ v
            size[i, g * group : (g + 1) * group] = w @ v.abs()
            most = max(most, k.shape[0])
            spread = max(spread, float((x.abs() @ k.abs().T).max()) * abs(scale))
    return out, size, most, spread
