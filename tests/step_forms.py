"""Definitions of the operators around a step with drafted tokens, in plain Python and
float64 numpy, with bounds on the kernels' errors where results are rounded.  States,
batches and masks as include/ipus.h describes them; nothing here calls the library."""
from __future__ import annotations

from collections import Counter

import numpy as np

from decoder_forms import HALF_STEP, SMALLEST


def tree(rng, rows, unused=0.0):
    """Masks (Python integers) of a random tree: row 0 its root, each row's parent one
    before it; with probability `unused` a row has none, not even itself."""
    masks = []
    for j in range(rows):
        parent = masks[rng.integers(0, j)] if j else 0
        masks.append(0 if j and rng.random() < unused else parent | 1 << j)
    return masks


def words(masks, count):
    """uint32 [rows][count]."""
    return np.array([[m >> 32 * w & 0xffffffff for w in range(count)] for m in masks],
                    np.uint32).reshape(len(masks), count)


# ---------------------------------------------------------------------------
def table_state(free, rows, pages, columns, missing=0):
    """The operator's int32 state of a list of free pages and of each sequence's pages."""
    table = np.full((len(rows), columns), -1, np.int32)
    for i, row in enumerate(rows):
        table[i, :len(row)] = row
    spare = list(free) + [-1] * (pages - len(free))
    return np.concatenate([[len(free), missing], spare, [len(r) for r in rows], table.ravel()]).astype(np.int32)


def fit_tables(free, rows, source, lengths, page_rows, columns):
    """(free, rows, missing) after the step."""
    need = [min(columns, -(-max(x, 0) // page_rows)) for x in lengths]
    mine = {}
    for i, p in enumerate(source):
        if 0 <= p < len(rows) and p not in mine.values():
            mine[i] = p
    kept = [0] * len(rows)
    for i, p in mine.items():
        kept[p] = min(len(rows[p]), need[i])
    free = list(free)
    for p, row in enumerate(rows):
        free += row[kept[p]:]
    out, missing = [], 0
    for i, n in enumerate(need):
        row = rows[mine[i]][:n] if i in mine else []
        while len(row) < n and free:
            row.append(free.pop())
        missing += n - len(row)
        out.append(row)
    return free, out, missing


def slot_maps(counts, lengths, table, rows, page_rows, pages, masks=None):
    """int32 [sequences + 1], [rows], [rows] one after the other."""
    offsets = [0]
    for n in counts:
        offsets.append(min(rows, offsets[-1] + max(n, 0)))
    position, slot = [0] * rows, [-1] * rows
    for s in range(len(counts)):
        n = offsets[s + 1] - offsets[s]
        for i in range(n):
            row, place = offsets[s] + i, lengths[s] - n + i
            p = place
            if masks is not None:
                p = lengths[s] - n + sum(masks[row] >> j & 1 for j in range(n) if j != i)
            position[row] = max(p, -1)
            if 0 <= place // page_rows < table.shape[1] and 0 <= table[s][place // page_rows] < pages:
                slot[row] = int(table[s][place // page_rows]) * page_rows + place % page_rows
    return np.array(offsets + position + slot, np.int64).astype(np.int32)


def keep_rows(caches, batch, path, counts):
    """[layers, pages, 2, heads, page rows, width] after the accepted rows have moved."""
    out, pr = caches.copy(), batch.page_rows

    def place(s, position):
        if position < 0 or position >= batch.lengths[s] or position // pr >= batch.columns:
            return None
        page = batch.table[s, position // pr]
        return (page, position % pr) if 0 <= page < batch.pages else None
    for s in range(batch.sequences()):
        n = int(batch.offsets[s + 1]) - int(batch.offsets[s])
        base, last = int(batch.lengths[s]) - n, -1
        for i in range(min(int(counts[s]), path.shape[1])):
            j = int(path[s, i])
            if not last < j < n:
                break
            last = j
            a, b = place(s, base + j), place(s, base + i)
            if j != i and a and b:
                out[:, b[0], :, :, b[1]] = out[:, a[0], :, :, a[1]]
    return out


# ---------------------------------------------------------------------------
def tree_attention(batch, masks, query, cache, key_heads, scale, fp16_probabilities=True):
    """As decoder_forms.attention, for rows that read the keys before their sequence's
    rows and those of the rows that their masks name.  The same bounds."""
    rows, heads, width = query.shape
    out, bound = np.zeros_like(query), np.zeros_like(query)
    inside = np.zeros(rows, bool)
    for s in range(batch.sequences()):
        first, n = int(batch.offsets[s]), batch.n[s]
        inside[first:first + n] = True
        p, page, row = batch.places(s)
        good = (page >= 0) & (page < batch.pages)
        p, page, row = p[good], page[good], row[good]
        if n == 0 or len(p) == 0:
            continue
        j = p - (batch.k[s] - n)  # of the sequence's rows; negative before them
        ok = np.array([[x < 0 or bool(masks[first + i] >> int(x) & 1) for x in j] for i in range(n)])
        for h in range(heads):
            kh = h // (heads // key_heads)
            k, v = cache[page, 0, kh, row], cache[page, 1, kh, row]
            q = query[first:first + n, h]
            with np.errstate(invalid="ignore"):
                x = (q @ k.T) * scale
                dx = (np.abs(q) @ np.abs(k).T) * scale * (width + 4) * 2.0 ** -24 + np.abs(x) * 2.0 ** -21
            x, dx = np.where(ok, x, -np.inf), np.where(ok, dx, 0.0)
            top = x.max(axis=1, keepdims=True)
            w = np.where(ok, np.exp(x - np.where(np.isfinite(top), top, 0.0)), 0.0)
            total = w.sum(axis=1, keepdims=True)
            w = np.where(total > 0, w / np.where(total > 0, total, 1.0), 0.0)
            at = slice(first, first + n)
            if np.all(np.isfinite(v)):
                out[at, h] = w @ v
            else:
                for r in range(n):
                    out[first + r, h] = w[r, ok[r]] @ v[ok[r]]
                v = np.where(np.isfinite(v), v, 0.0)
            step = 2 * 2.0 ** -11 if fp16_probabilities else 0.0
            tiny = 2.0 ** -17 if fp16_probabilities else 0.0
            delta = 2.0 * dx.max(axis=1, keepdims=True)
            bound[at, h] = ((step + delta + len(p) * 2.0 ** -23) * (w @ np.abs(v))
                            + tiny * (ok @ np.abs(v)) / np.maximum(total, 1.0))
    return out, bound, inside


# ---------------------------------------------------------------------------
def adjust_logits(x, offsets, tokens, masks, history, counts, penalties, bias_offsets, biases, allowed):
    """x [rows, columns] in float64 after penalties, biases and masks; the bound before
    the last rounding; which rows belong to a sequence.  masks: Python integers, or None
    for rows in order; allowed: truth values [rows, columns], or None."""
    rows, columns = x.shape
    out, bound, inside = x.copy(), np.zeros_like(x), np.zeros(rows, bool)
    step = 2.0 ** -24
    for s in range(len(offsets) - 1):
        first, end = int(offsets[s]), int(offsets[s + 1])
        prompt, total = int(counts[s][0]), int(counts[s][1])
        total = min(max(total, 0), history.shape[1])
        prompt = min(max(prompt, 0), total)
        r, f, p = (float(t) for t in penalties[s])
        bias = {}
        for e in range(int(bias_offsets[s]), int(bias_offsets[s + 1])):
            bias[int(biases[0][e])] = float(biases[1][e])  # the last entry of a token
        for row in range(first, end):
            inside[row] = True
            made = Counter(int(t) for t in history[s, prompt:total])
            for j in range(end - first):
                if (masks[row] >> j & 1) if masks is not None else j <= row - first:
                    made[int(tokens[first + j])] += 1
            for t in sorted(set(made) | {int(t) for t in history[s, :prompt]}):
                if not 0 <= t < columns:
                    continue
                y = out[row, t]
                y = y / r if y > 0 else y * r
                e = abs(y) * step  # each product, sum and difference rounded in fp32
                if made[t]:
                    z = f * made[t] + p
                    y, e = y - z, e + abs(z) * 2 * step
                    e += abs(y) * step
                out[row, t], bound[row, t] = y, e
            for t, b in bias.items():
                if 0 <= t < columns:
                    out[row, t] += b
                    bound[row, t] += (abs(out[row, t]) + bound[row, t]) * step
            if allowed is not None:
                out[row] = np.where(allowed[row], out[row], -np.inf)
    return out, bound, inside


def within(got, want, bound, dtype):
    """Whether each element is its value, rounded once to `dtype`, within the bound before
    that; infinities and NaN in their places."""
    got = got.astype(np.float64)
    finite = np.isfinite(want)
    same = np.where(np.isnan(want), np.isnan(got), got == want)
    with np.errstate(invalid="ignore"):
        near = np.abs(got - want) <= bound + (np.abs(want) + bound) * HALF_STEP[dtype] + SMALLEST[dtype]
    return np.where(finite, near, same)
