"""The operators of a decoder's step with drafted tokens as programs run them on
one MI355X: page tables fitted to the requests' lengths, row offsets, positions
and cache slots of the step's rows, attention of trees of drafted tokens over the
paged cache, penalties, biases and grammar masks on their logits, and the removal
of the rejected drafts from the cache.

Each case is a dict of plain values; `prepare` makes its inputs on the GPU and
what a program keeps between calls, `run` is one pass: through the kernel ABI
where `own` is true, in elementary torch operations where it is false.  `exact` is
the operator's definition in 64 bits, one sequence and row after the other.

The cache is [pages][2][key heads][page rows][width] fp16, keys before values;
row p of sequence s lies in page table[s][p / page_rows] at row p % page_rows.
Rows offsets[s] .. offsets[s + 1] - 1 of a step belong to sequence s, the last of
them at position lengths[s] - 1.  Bit j of a row's mask says that it reads the j-th
row of its sequence: of a tree, its ancestors and itself.
"""
import math
import random
import struct
from collections import Counter

import torch

own = False

F16, F32, F64, I32 = torch.float16, torch.float32, torch.float64, torch.int32

_CONTEXT = None


def _context():
    """The program's one device context, kept for its whole run."""
    global _CONTEXT
    if _CONTEXT is None:
        import __graft_entry__
        _CONTEXT = __graft_entry__.import_package().Context(0)
    return _CONTEXT


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def tables(sequences, columns, page_rows, step, turnover, spare, pattern):
    """Sequences of up to `columns` pages that grow by up to `step` tokens or
    lose some (rejected drafts); of 1000, `turnover` have ended and others begin
    in their place.  `spare` pages are free before the step."""
    return {"kind": "tables", "sequences": sequences, "columns": columns, "page_rows": page_rows,
            "step": step, "turnover": turnover, "spare": spare, "pattern": pattern}


def slots(sequences, rows, keys, page_rows, tree, padding, pattern):
    """Up to `rows` new rows of each sequence, whose length with them is up to
    `keys`; as a tree, or one after the other; `padding` rows behind the last."""
    return {"kind": "slots", "sequences": sequences, "rows": rows, "keys": keys,
            "page_rows": page_rows, "tree": tree, "padding": padding, "pattern": pattern}


def attention(sequences, nodes, keys, query_heads, key_heads, width, page_rows, batch, holes,
              pattern, padding):
    """Trees of `nodes` drafted tokens: of all sequences ("equal", against `keys`
    keys), or nodes / 2 .. nodes against keys / 16 .. keys ("ragged").  With `holes` some
    rows of a tree stay unused: their masks are empty."""
    return {"kind": "attention", "sequences": sequences, "rows": nodes, "keys": keys,
            "query_heads": query_heads, "key_heads": key_heads, "width": width,
            "page_rows": page_rows, "batch": batch, "holes": holes, "tree": True,
            "pattern": pattern, "padding": padding}


def logits(sequences, nodes, columns, f32, tree, history, biases, grammar, pattern, padding):
    """Logits of up to `nodes` rows of each sequence, behind up to `history`
    tokens, up to `biases` biased ones each; with `grammar` a row's tokens are
    those that its mask allows (few, most, or all of them)."""
    return {"kind": "logits", "sequences": sequences, "rows": nodes, "columns": columns, "f32": f32,
            "tree": tree, "history": history, "biases": biases, "grammar": grammar,
            "pattern": pattern, "padding": padding}


def keep(sequences, nodes, kept, keys, layers, key_heads, width, page_rows, pattern):
    """Up to `kept` of `nodes` drafted tokens stay, in the caches of all layers."""
    return {"kind": "keep", "sequences": sequences, "rows": nodes, "kept": kept, "keys": keys,
            "layers": layers, "key_heads": key_heads, "width": width, "page_rows": page_rows,
            "tree": True, "batch": "ragged", "padding": 0, "pattern": pattern}


def listed():
    return [
        # One step of a decoding batch: each sequence grows by a token, a few
        # need a page.  The launch is everything.
        dict(tables(64, 256, 16, 1, 0, 500, 1), name="tables_decode"),
        # A large batch of long contexts between steps: an eighth of the requests
        # ended, new prompts begin, drafts were rejected.
        dict(tables(512, 2048, 16, 64, 125, 100000, 2), name="tables_turnover"),
        # One token of each of 64 sequences.
        dict(slots(64, 1, 4096, 16, False, 0, 3), name="slots_decode"),
        # 1000 sequences' trees of up to 64 drafts, padded at the end.
        dict(slots(1000, 64, 2000, 16, True, 37, 4), name="slots_trees"),
        # The smallest verification: 4 sequences, 8 drafts each.
        dict(attention(4, 8, 1024, 16, 16, 64, 16, "ragged", False, 5, 0), name="tree_small"),
        # A serving step: 64 sequences of very different lengths, 4 drafts each.
        dict(attention(64, 4, 32768, 32, 8, 128, 64, "ragged", False, 6, 0), name="tree_ragged"),
        # Wide trees: 16 sequences verify 64 drafts each.
        dict(attention(16, 64, 8192, 32, 8, 128, 64, "equal", False, 7, 0), name="tree_wide"),
        # Odd sizes, masks of unused rows, padded.
        dict(attention(7, 99, 3001, 16, 16, 72, 32, "ragged", True, 8, 5), name="tree_odd"),
        # Logits of a decoding step: 64 rows, an odd vocabulary, no grammar.
        dict(logits(64, 1, 50001, False, False, 1000, 20, False, 9, 0), name="logits_decode"),
        # Logits of 64 trees of 16 drafts in fp32, with everything.
        dict(logits(64, 16, 131072, True, True, 8192, 300, True, 10, 0), name="logits_trees"),
        # One layer's cache of 8 sequences after a verification.
        dict(keep(8, 8, 4, 1024, 1, 8, 128, 16, 11), name="keep_small"),
        # All of 16 layers, 64 sequences, up to 12 of 64 drafts each.
        dict(keep(64, 64, 12, 512, 16, 8, 128, 64, 12), name="keep_layers"),
    ]


def _log_size(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the same ranges: a kind, then sizes over its range."""
    kind = rng.choice(["tables", "slots", "attention", "attention", "logits", "logits", "keep"])
    page_rows, pattern = rng.choice([8, 16, 16, 32, 64, 128]), rng.randrange(1 << 20)
    padding = rng.choice([0, 0, rng.randint(1, 100)])
    if kind == "tables":
        while True:
            sequences, columns = _log_size(rng, 1, 2048), _log_size(rng, 1, 4096)
            if sequences * columns <= 512 * 2048:
                break
        return tables(sequences, columns, page_rows, _log_size(rng, 1, 4096),
                      rng.choice([0, 0, 50, 500]), _log_size(rng, 1, 100000), pattern)
    if kind == "slots":
        while True:
            sequences, rows = _log_size(rng, 1, 2048), _log_size(rng, 1, 8192)
            keys = max(rows, _log_size(rng, 1, 32768))
            if sequences * rows <= 64000 and sequences * keys <= 1 << 24:
                break
        return slots(sequences, rows, keys, page_rows, rows <= 256 and rng.random() < 0.6, padding,
                     pattern)
    width = rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 128, 192, 256])
    key_heads, group = rng.choice([(16, 1), (12, 1), (8, 4), (8, 8), (4, 4), (2, 7), (1, 16)])
    if kind == "attention":
        while True:
            sequences, nodes = _log_size(rng, 1, 128), _log_size(rng, 1, 256)
            keys = max(nodes, _log_size(rng, 1, 32768))
            if (sequences * keys * key_heads * width <= 64 * 16384 * 8 * 128
                    and sequences * nodes * keys * key_heads * group * width
                    <= 16 * 64 * 8192 * 32 * 128):
                break
        return attention(sequences, nodes, keys, key_heads * group, key_heads, width, page_rows,
                         rng.choice(["equal", "ragged"]), rng.random() < 0.3, pattern, padding)
    if kind == "logits":
        while True:
            sequences, nodes = _log_size(rng, 1, 256), rng.choice([1, 1, _log_size(rng, 2, 64)])
            columns = _log_size(rng, 100, 262144)
            if sequences * nodes * columns <= 64 * 16 * 131072:
                break
        return logits(sequences, nodes, columns, rng.random() < 0.5, rng.random() < 0.6,
                      rng.choice([0, _log_size(rng, 1, 8192)]),
                      rng.choice([0, _log_size(rng, 1, 300)]),
                      rng.random() < 0.5, pattern, padding)
    while True:
        sequences, nodes = _log_size(rng, 1, 128), _log_size(rng, 1, 128)
        keys, layers = max(nodes, _log_size(rng, 1, 4096)), _log_size(rng, 1, 32)
        if sequences * keys * layers * key_heads * width <= 64 * 512 * 16 * 8 * 128:
            break
    return keep(sequences, nodes, rng.randint(1, nodes), keys, layers, key_heads, width, page_rows,
                pattern)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed, tensor):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 16 + tensor)
    return g


def _normal(seed, tensor, shape, dtype, scale=1.0):
    x = torch.randn(shape, generator=_generator(seed, tensor), device="cuda", dtype=F32)
    return x.mul_(scale).to(dtype)


def _uniform(seed, tensor, shape, low, high):
    x = torch.rand(shape, generator=_generator(seed, tensor), device="cuda", dtype=F32)
    return x.mul_(high - low).add_(low)


def _ints(values, shape=None):
    x = torch.tensor(values, dtype=I32, device="cuda")
    return x if shape is None else x.reshape(shape)


def _words(masks, words):
    """Python integers as rows of `words` 32-bit words."""
    data = b"".join(m.to_bytes(4 * words, "little") for m in masks)
    return torch.frombuffer(bytearray(data), dtype=I32).reshape(len(masks), words).to("cuda")


def _batch(c):
    """New rows and lengths of the sequences, of the case alone."""
    rng = random.Random(c["pattern"])
    n, k = [], []
    for _ in range(c["sequences"]):
        if c.get("batch") == "equal":
            n.append(c["rows"])
            k.append(c["keys"])
        else:
            n.append(rng.randint(max(1, c["rows"] // 2), c["rows"]))
            if "keys" in c:
                k.append(max(n[-1], _log_size(rng, max(1, c["keys"] // 16), c["keys"])))
    return n, k


def _trees(c, seed, n):
    """Every sequence's masks: row 0 is the last token chosen, each later row's
    parent an earlier one (with `holes`, some rows stay unused)."""
    rng = random.Random(c["pattern"] * 1000003 + seed)
    masks = []
    for rows in n:
        mine = []
        for j in range(rows):
            parent = mine[rng.randrange(max(0, j - 12), j)] if j else 0
            unused = c.get("holes") and j and rng.random() < 0.1
            mine.append(0 if unused else parent | 1 << j)
        masks += mine
    return masks


def _mask_words(c):
    return (c["rows"] + 31) // 32 if c["tree"] else 0


def _paged(c, seed):
    """Offsets, lengths, masks and a table of pages in no order, entries past a
    sequence's end -1."""
    n, k = _batch(c)
    pr = c["page_rows"]
    need = [(x + pr - 1) // pr for x in k]
    columns, pages = max(need) + 2, sum(need) + 3
    order = torch.randperm(pages, generator=_generator(seed, 9), device="cuda", dtype=torch.int64)
    held = _ints(need).long()
    start, column = held.cumsum(0) - held, torch.arange(columns, device="cuda")[None, :]
    entry = order[(start[:, None] + column).clamp_(max=pages - 1)]
    table = torch.where(column < held[:, None], entry, -1).to(I32)
    offsets = [0]
    for x in n:
        offsets.append(offsets[-1] + x)
    words = _mask_words(c)
    rows = offsets[-1] + c["padding"]
    masks = _trees(c, seed, n) + [0] * c["padding"] if words else []
    return {"n": n, "k": k, "columns": columns, "pages": pages, "rows": rows, "table": table,
            "offsets": offsets, "row_offsets": _ints(offsets), "lengths": _ints(k),
            "counts": _ints(n), "masks": masks, "words": words,
            "mask": _words(masks, words) if words else _ints([[0]])}


def _requests(c, seed):
    """Lengths before the step, the sequences' places in the last one, and lengths
    to be: pages go by these."""
    rng = random.Random(c["pattern"] * 1000003 + seed)
    most = c["columns"] * c["page_rows"]
    before = [_log_size(rng, max(1, most // 16), most) for _ in range(c["sequences"])]
    source, lengths = list(range(c["sequences"])), []
    if c["turnover"]:
        rng.shuffle(source)
    for i, s in enumerate(source):
        if rng.randrange(1000) < c["turnover"]:
            source[i] = -1
            lengths.append(_log_size(rng, 1, most))
        else:
            change = rng.randint(1, c["step"]) - (rng.randint(0, c["step"]) if c["step"] > 1 else 0)
            lengths.append(max(1, min(most, before[s] + change)))
    return before, source, lengths


def _prepare_tables(c, seed, state):
    before, source, lengths = _requests(c, seed)
    pr, columns, count = c["page_rows"], c["columns"], c["sequences"]
    held = [(x + pr - 1) // pr for x in before]
    used = sum(held)
    # The same number of pages for inputs of any seed, as a server's.
    pages = max(used, count * columns // 2) + c["spare"]
    order = torch.randperm(pages, generator=_generator(seed, 1), device="cuda", dtype=torch.int64)
    h = _ints(held).long()
    start, column = h.cumsum(0) - h, torch.arange(columns, device="cuda")[None, :]
    entry = order[(start[:, None] + column).clamp_(max=pages - 1)]
    table = torch.where(column < h[:, None], entry, -1)
    free = torch.full((pages,), -1, dtype=torch.int64, device="cuda")
    free[:pages - used] = order[used:]
    head = torch.tensor([pages - used, 0], device="cuda")
    state["previous"] = torch.cat([head, free, h, table.flatten()]).to(I32)
    state["source"], state["lengths"] = _ints(source), _ints(lengths)
    state["pages"] = pages
    state["out"] = torch.empty(2 + pages + count * (1 + columns), dtype=I32, device="cuda")


def _prepare_logits(c, seed, state):
    n, _ = _batch(c)
    rng = random.Random(c["pattern"] * 1000003 + seed + 1)
    columns, dtype = c["columns"], F32 if c["f32"] else F16
    offsets = [0]
    for x in n:
        offsets.append(offsets[-1] + x)
    rows, words = offsets[-1] + c["padding"], _mask_words(c)
    state.update(n=n, offsets=offsets, rows=rows, words=words, row_offsets=_ints(offsets))
    state["masks"] = _trees(c, seed, n) + [0] * c["padding"] if words else []
    state["mask"] = _words(state["masks"], words) if words else _ints([[0]])
    state["x"] = _normal(seed, 1, (rows, columns), dtype, 3.0)
    state["out"] = torch.zeros((rows, columns), dtype=dtype, device="cuda")
    # Texts repeat: half of their tokens are of the first few hundred.
    few = min(columns, 400)

    def tokens(tensor, shape):
        any_token = (_uniform(seed, tensor, shape, 0, 1) * columns).to(I32).clamp_(max=columns - 1)
        common = (_uniform(seed, tensor + 1, shape, 0, 1) * few).to(I32).clamp_(max=few - 1)
        return torch.where(_uniform(seed, tensor + 2, shape, 0, 1) < 0.5, any_token, common)
    state["tokens"] = tokens(2, (rows,))
    width = max(1, c["history"])
    state["history"] = tokens(5, (c["sequences"], width))
    counts = []
    for _ in n:
        total = rng.randint(c["history"] // 2, c["history"])
        counts.append([rng.randint(0, total), total])
    state["history_counts"] = _ints(counts)
    repetition, others = _uniform(seed, 8, (len(n), 1), 1.0, 1.3), _uniform(seed, 9, (len(n), 2), 0.0, 0.5)
    state["penalties"] = torch.cat([repetition, others], dim=1).contiguous()
    begin, entries = [0], []
    for _ in n:
        mine = rng.sample(range(columns), min(columns, rng.randint(c["biases"] // 2, c["biases"])))
        entries += [[t, struct.unpack("<i", struct.pack("<f", rng.uniform(-5.0, 5.0)))[0]] for t in mine]
        begin.append(len(entries))
    state["bias_offsets"], state["bias_count"] = _ints(begin), len(entries)
    state["biases"] = _ints(entries or [[0, 0]])
    if c["grammar"]:
        # A token in 64, half of them, or all of a row's.
        shape = (rows, (columns + 31) // 32)
        bits = [torch.randint(-1 << 31, 1 << 31, shape, generator=_generator(seed, 10 + i), device="cuda")
                for i in range(6)]
        few_bits = bits[0]
        for b in bits[1:]:
            few_bits = few_bits & b
        pick = torch.arange(rows, device="cuda")[:, None] % 3
        state["allowed"] = torch.where(pick == 0, few_bits, torch.where(pick == 1, bits[0], -1)).to(I32)
    else:
        state["allowed"] = _ints([[0]])


def prepare(case, seed):
    c = case
    state = {"case": c}
    if c["kind"] == "tables":
        _prepare_tables(c, seed, state)
    elif c["kind"] == "logits":
        _prepare_logits(c, seed, state)
    else:
        state.update(_paged(c, seed))
    if c["kind"] == "slots":
        state["out"] = torch.empty(c["sequences"] + 1 + 2 * state["rows"], dtype=I32, device="cuda")
    if c["kind"] == "attention":
        pool = (state["pages"], 2, c["key_heads"], c["page_rows"], c["width"])
        state["cache"] = _normal(seed, 1, pool, F16)
        heads = (state["rows"], c["query_heads"], c["width"])
        state["q"] = _normal(seed, 2, heads, F16, 1.5)
        state["out"] = torch.zeros(heads, dtype=F16, device="cuda")
    if c["kind"] == "keep":
        pool = (c["layers"], state["pages"], 2, c["key_heads"], c["page_rows"], c["width"])
        state["cache"] = _normal(seed, 1, pool, F16)
        state["paths"] = _paths(c, seed, state["n"])
        state["path"] = _ints([p + [-1] * (c["kept"] - len(p)) for p in state["paths"]])
        state["path_counts"] = _ints([len(p) for p in state["paths"]])
    # What a program keeps for its launches: the addresses and sizes.
    state["call"] = _call(state)
    # The inputs were made on torch's stream, the library has its own.
    torch.cuda.synchronize()
    return state


def _paths(c, seed, n):
    """The accepted rows of each tree: the root and some of the others, in order."""
    rng = random.Random(c["pattern"] * 1000003 + seed + 2)
    paths = []
    for rows in n:
        count = rng.randint(1, min(rows, c["kept"]))
        paths.append([0] + sorted(rng.sample(range(1, rows), count - 1)))
    return paths


def _call(state):
    """Symbol, output, inputs and scalars of the case's launch."""
    c, s = state["case"], state
    if c["kind"] == "tables":
        return ("ipu_stack_page_tables", s["out"].data_ptr(),
                [s[t].data_ptr() for t in ("previous", "source", "lengths")],
                [c["sequences"], c["sequences"], s["pages"], c["page_rows"], c["columns"]])
    if c["kind"] == "slots":
        return ("ipu_stack_slot_maps", s["out"].data_ptr(),
                [s[t].data_ptr() for t in ("counts", "lengths", "table", "mask")],
                [c["sequences"], s["rows"], s["pages"], c["page_rows"], s["columns"], s["words"]])
    if c["kind"] == "attention":
        return ("ipu_stack_attention_tree_pages_f16", s["out"].data_ptr(),
                [s[t].data_ptr() for t in ("q", "cache", "table", "row_offsets", "lengths", "mask")],
                [c["sequences"], s["rows"], max(s["n"]), c["query_heads"], c["key_heads"],
                 c["width"], c["query_heads"] * c["width"], s["pages"], c["page_rows"],
                 s["columns"], s["words"], 0])
    if c["kind"] == "logits":
        return ("ipu_stack_adjust_logits_f32" if c["f32"] else "ipu_stack_adjust_logits_f16",
                s["out"].data_ptr(),
                [s[t].data_ptr() for t in ("x", "row_offsets", "tokens", "mask", "history",
                                           "history_counts", "penalties", "bias_offsets",
                                           "biases", "allowed")],
                [c["sequences"], s["rows"], c["columns"], c["columns"], c["columns"], s["words"],
                 c["history"], s["bias_count"], s["allowed"].shape[1] if c["grammar"] else 0])
    return ("ipu_stack_keep_pages_f16", s["cache"].data_ptr(),
            [s[t].data_ptr() for t in ("table", "row_offsets", "lengths", "path", "path_counts")],
            [c["sequences"], s["rows"], c["layers"], c["key_heads"], c["width"], s["pages"],
             c["page_rows"], s["columns"], c["kept"]])


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        _context().launch(*state["call"])
        return state["cache"] if state["case"]["kind"] == "keep" else state["out"]
    return _PLAIN[state["case"]["kind"]](state)


def _plain_tables(s):
    c, pages = s["case"], s["pages"]
    count, columns, device = c["sequences"], c["columns"], "cuda"
    previous = s["previous"].long()
    free, spare = previous[0], previous[2:2 + pages]
    held = previous[2 + pages:2 + pages + count]
    old = previous[2 + pages + count:].view(count, columns)
    source, place = s["source"].long(), torch.arange(count, device=device)
    need = ((s["lengths"].long() + c["page_rows"] - 1) // c["page_rows"]).clamp(0, columns)
    valid = (source >= 0) & (source < count)
    # The first sequence that names a row goes on with it.
    owner = torch.full((count + 1,), count, device=device)
    owner.scatter_reduce_(0, torch.where(valid, source, count), place, "amin")
    at = source.clamp(0, count - 1)
    base = torch.where(valid & (owner[at] == place), held[at], 0)
    kept = torch.minimum(base, need)
    # Pages given back, behind the free ones.
    owner = owner[:count]
    stays = torch.where(owner < count, kept[owner.clamp(max=count - 1)], 0)
    column = torch.arange(columns, device=device)[None, :]
    back = ((column >= stays[:, None]) & (column < held[:, None])).flatten()
    listed_pages = torch.cat([spare, spare[:1]])
    listed_pages.scatter_(0, torch.where(back, free + back.cumsum(0) - 1, pages),
                          old.flatten())
    total = free + back.sum()
    # Pages taken, from the end.
    want = need - kept
    begin = want.cumsum(0) - want
    got = torch.minimum((total - begin).clamp(min=0), want)
    take = (total - 1 - begin[:, None] - (column - kept[:, None])).clamp(0, pages - 1)
    table = torch.where(column < (kept + got)[:, None], listed_pages[take], -1)
    table = torch.where(column < kept[:, None], old[at], table)
    left = total - got.sum()
    rest = torch.where(torch.arange(pages, device=device) < left, listed_pages[:pages], -1)
    head = torch.stack([left, (want - got).sum()])
    return s["out"].copy_(torch.cat([head, rest, kept + got, table.flatten()]))


def _bits_of(words):
    """[rows][words] -> truth values [rows][32 words]."""
    shift = torch.arange(32, dtype=I32, device="cuda")
    return ((words[:, :, None] >> shift) & 1).flatten(1) != 0


def _plain_slots(s):
    c, rows = s["case"], s["rows"]
    offsets = torch.cat([s["counts"].new_zeros(1), s["counts"].cumsum(0)]).long()
    row = torch.arange(rows, device="cuda")
    sequence = torch.searchsorted(offsets[1:], row, right=True)
    inside = sequence < c["sequences"]
    sequence = sequence.clamp(max=c["sequences"] - 1)
    n, first = s["counts"][sequence].long(), offsets[sequence]
    base = s["lengths"][sequence].long() - n
    place = base + row - first
    position = place
    if s["words"]:
        bits = _bits_of(s["mask"])
        j = torch.arange(bits.shape[1], device="cuda")[None, :]
        others = bits & (j < n[:, None]) & (j != (row - first)[:, None])
        position = base + others.sum(dim=1)
    page = s["table"][sequence, (place // c["page_rows"]).clamp(0, s["columns"] - 1)].long()
    good = inside & (place >= 0) & (place < s["columns"] * c["page_rows"]) & (page >= 0)
    slot = torch.where(good, page * c["page_rows"] + place % c["page_rows"], -1)
    position = torch.where(inside & (position >= 0), position, torch.where(inside, -1, 0))
    return s["out"].copy_(torch.cat([offsets, position, slot]))


def _plain_attention(s):
    c = s["case"]
    heads, width, count = c["key_heads"], c["width"], c["sequences"]
    group, most = c["query_heads"] // heads, c["rows"]
    keys = max(s["k"])
    # All sequences as long as the longest: what lies behind a sequence's end
    # has no weight.
    used = (keys + c["page_rows"] - 1) // c["page_rows"]
    pages = s["cache"][s["table"][:, :used].clamp(min=0).long()]
    kv = pages.permute(2, 0, 3, 1, 4, 5).reshape(2, count, heads, -1, width)[:, :, :, :keys].to(F32)
    node = torch.arange(most, device="cuda")[None, :]
    real = node < s["counts"][:, None]
    row = torch.where(real, s["row_offsets"][:-1, None] + node, 0).long()
    q = s["q"][row].to(F32).reshape(count, most, heads, group, width).permute(0, 2, 1, 3, 4)
    x = torch.matmul(q.reshape(count, heads, most * group, width),
                     kv[0].transpose(2, 3).contiguous()).mul_(width ** -0.5)
    # Keys before the new rows, and those of the mask.
    base = (s["lengths"] - s["counts"])[:, None, None]
    key = torch.arange(keys, device="cuda")[None, None, :]
    bits = _bits_of(s["mask"])[row]  # [sequences][rows][bits]
    drafted = (key - base).clamp(0, bits.shape[2] - 1).long().expand(-1, most, -1)
    seen = (key < base) | (torch.gather(bits, 2, drafted) & (key < s["lengths"][:, None, None]))
    x = x.reshape(count, heads, most, group, keys)
    x = x.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = x.amax(dim=4, keepdim=True)
    p = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    y = torch.matmul(p.reshape(count, heads, most * group, keys), kv[1])
    total = p.sum(dim=4, keepdim=True)
    y = y.reshape(count, heads, most, group, width) / torch.where(total == 0.0, 1.0, total)
    y = y.permute(0, 2, 1, 3, 4).reshape(count * most, heads * group, width)
    s["out"][row[real]] = y[real.flatten()].to(F16)
    return s["out"]


def _plain_logits(s):
    c, rows, columns = s["case"], s["rows"], s["case"]["columns"]
    row = torch.arange(rows, device="cuda")
    sequence = torch.searchsorted(s["row_offsets"][1:], row, right=True)
    sequence = sequence.clamp(max=c["sequences"] - 1)
    # How often a token stands in the prompt and behind it; one more column
    # takes what does not count.
    step = torch.arange(s["history"].shape[1], device="cuda")[None, :]
    prompt, total = s["history_counts"][:, :1], s["history_counts"][:, 1:]
    ones = torch.ones_like(s["history"], dtype=F32)
    seen, made = (torch.zeros((c["sequences"], columns + 1), device="cuda").scatter_add_(
        1, torch.where(part, s["history"], columns).long(), ones)
        for part in (step < prompt, (step >= prompt) & (step < total)))
    # The row's path: itself and the rows that its mask, or their order, says.
    first = s["row_offsets"][sequence].long()
    n = s["row_offsets"][sequence + 1].long() - first
    j = torch.arange(max(32 * s["words"], c["rows"]), device="cuda")[None, :]
    if s["words"]:
        path = _bits_of(s["mask"])
        j = j[:, :path.shape[1]]
        path = path & (j < n[:, None])
    else:
        path = j <= (row - first)[:, None]
    token = s["tokens"][(first[:, None] + j).clamp(max=rows - 1)]
    made = made[sequence].scatter_add_(1, torch.where(path, token, columns).long(),
                                       torch.ones(path.shape, device="cuda"))[:, :columns]
    seen = seen[sequence][:, :columns] + made
    repetition, frequency, presence = (s["penalties"][sequence, i:i + 1] for i in range(3))
    x = s["x"].to(F32)
    x = torch.where(seen > 0, torch.where(x > 0, x / repetition, x * repetition), x)
    x = x - frequency * made - presence * (made > 0)
    if s["bias_count"]:
        entry = torch.arange(s["bias_count"], device="cuda")
        owner = torch.searchsorted(s["bias_offsets"][1:], entry, right=True)
        bias = torch.zeros((c["sequences"], columns), device="cuda")
        bias[owner, s["biases"][:, 0].long()] = s["biases"][:, 1].contiguous().view(F32)
        x = x + bias[sequence]
    if c["grammar"]:
        x = torch.where(_bits_of(s["allowed"])[:, :columns], x, -math.inf)
    used = s["offsets"][-1]
    s["out"][:used] = x[:used].to(s["out"].dtype)
    return s["out"]


def _plain_keep(s):
    c, pr = s["case"], s["case"]["page_rows"]
    step = torch.arange(c["kept"], device="cuda")[None, :]
    sequence = torch.arange(c["sequences"], device="cuda")[:, None]
    base = (s["lengths"] - s["counts"])[:, None]
    moves = (step < s["path_counts"][:, None]) & (s["path"] != step)
    source, to = (base + s["path"])[moves].long(), (base + step)[moves].long()
    sequence = sequence.expand(-1, c["kept"])[moves]
    rows = s["cache"][:, s["table"][sequence, source // pr].long(), :, :, source % pr]
    s["cache"][:, s["table"][sequence, to // pr].long(), :, :, to % pr] = rows
    return s["cache"]


_PLAIN = {"tables": _plain_tables, "slots": _plain_slots, "attention": _plain_attention,
          "logits": _plain_logits, "keep": _plain_keep}


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its exact result
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "tables":
        # Of any seed, about: the pages that sequences hold, read and written,
        # and the free ones' list.
        before, _, lengths = _requests(c, 0)
        pr, total = c["page_rows"], c["sequences"] * c["columns"]
        held = sum((x + pr - 1) // pr for x in before)
        free = max(0, max(held, total // 2) - held) + c["spare"]
        return {"bytes": 4 * (held + total + 2 * free + 5 * c["sequences"]), "flops": 0}
    n, k = _batch(c)
    words = _mask_words(c)
    if c["kind"] == "slots":
        return {"bytes": 4 * (3 * len(n) + sum(n) * (3 + words)), "flops": 0}
    if c["kind"] == "logits":
        size = 4 if c["f32"] else 2
        bits = sum(n) * ((c["columns"] + 31) // 32) * 4 if c["grammar"] else 0
        lists = len(n) * (c["history"] * 3 // 4 * 4 + c["biases"] * 3 // 4 * 8 + 24)
        return {"bytes": 2 * sum(n) * c["columns"] * size + bits + lists + 4 * sum(n) * (1 + words),
                "flops": 0}
    if c["kind"] == "keep":
        moved = sum(sum(i != p for i, p in enumerate(path)) for path in _paths(c, 0, n))
        row = c["layers"] * 2 * c["key_heads"] * c["width"] * 2
        return {"bytes": 2 * moved * row + 4 * (3 + c["kept"]) * len(n), "flops": 0}
    table = sum((x + c["page_rows"] - 1) // c["page_rows"] for x in k)
    moved = 2 * 2 * (sum(k) * c["key_heads"] + sum(n) * c["query_heads"]) * c["width"]
    # The keys before the new rows, and about half a dozen of the tree's.
    pairs = sum(a * (b - a) + a * min(a, 6) for a, b in zip(n, k))
    return {"bytes": moved + 4 * (2 * len(n) + 1 + table + sum(n) * words),
            "flops": 4 * pairs * c["query_heads"] * c["width"]}


def exact(case, seed):
    s = {"case": case}
    if case["kind"] == "tables":
        _prepare_tables(case, seed, s)
    elif case["kind"] == "logits":
        _prepare_logits(case, seed, s)
    else:
        s.update(_paged(case, seed))
    return _EXACT[case["kind"]](case, seed, s)


def _exact_tables(c, seed, s):
    pages, count, columns = s["pages"], c["sequences"], c["columns"]
    previous = s["previous"].tolist()
    free = previous[2:2 + previous[0]]
    held, old = previous[2 + pages:2 + pages + count], previous[2 + pages + count:]
    rows = [old[i * columns:i * columns + h] for i, h in enumerate(held)]
    mine, kept = {}, [0] * count
    need = [min(columns, -(-x // c["page_rows"])) for x in s["lengths"].tolist()]
    for i, p in enumerate(s["source"].tolist()):
        if 0 <= p < count and p not in mine.values():
            mine[i] = p
            kept[p] = min(held[p], need[i])
    for p, row in enumerate(rows):
        free += row[kept[p]:]
    table, counts, missing = [], [], 0
    for i in range(count):
        row = rows[mine[i]][:need[i]] if i in mine else []
        while len(row) < need[i] and free:
            row.append(free.pop())
        missing += need[i] - len(row)
        counts.append(len(row))
        table += row + [-1] * (columns - len(row))
    return _ints([len(free), missing] + free + [-1] * (pages - len(free)) + counts + table)


def _exact_slots(c, seed, s):
    position, slot, pr = [], [], c["page_rows"]
    table = s["table"].tolist()
    for i, (n, k) in enumerate(zip(s["n"], s["k"])):
        for j in range(n):
            p = k - n + j
            slot.append(table[i][p // pr] * pr + p % pr)
            if s["words"]:
                p = k - n + (s["masks"][s["offsets"][i] + j] & ~(1 << j)).bit_count()
            position.append(p)
    rest = [0] * c["padding"]
    return _ints(s["offsets"] + position + rest + slot + [-1] * c["padding"])


def _exact_attention(c, seed, s):
    if work(c)["flops"] > 2.5e12:  # too long in 64 bits
        return None
    pool = (s["pages"], 2, c["key_heads"], c["page_rows"], c["width"])
    cache = _normal(seed, 1, pool, F16)
    q = _normal(seed, 2, (s["rows"], c["query_heads"], c["width"]), F16, 1.5)
    out = torch.zeros(q.shape, dtype=F64, device="cuda")
    group = c["query_heads"] // c["key_heads"]
    for i, (n, k) in enumerate(zip(s["n"], s["k"])):
        at = s["offsets"][i]
        place = torch.arange(k, device="cuda")
        page, row = s["table"][i].long()[place // c["page_rows"]], place % c["page_rows"]
        hidden = torch.zeros((n, k), dtype=torch.bool)
        for j in range(n):
            for m in range(n):
                hidden[j, k - n + m] = not s["masks"][at + j] >> m & 1
        hidden = hidden.to("cuda")
        for h in range(c["query_heads"]):
            key, value = (cache[page, x, h // group, row].to(F64) for x in (0, 1))
            x = torch.mm(q[at:at + n, h].to(F64), key.t().contiguous()) / math.sqrt(c["width"])
            weight = torch.softmax(x.masked_fill(hidden, -math.inf), dim=1)
            out[at:at + n, h] = torch.mm(torch.nan_to_num(weight), value)
    return out


def _exact_logits(c, seed, s):
    out = torch.zeros((s["rows"], c["columns"]), dtype=F64, device="cuda")
    history, counts = s["history"].tolist(), s["history_counts"].tolist()
    tokens, penalties = s["tokens"].tolist(), s["penalties"].tolist()
    biases, begin = s["biases"].tolist(), s["bias_offsets"].tolist()
    shift = torch.arange(32, device="cuda")
    for i, n in enumerate(s["n"]):
        first, (prompt, total) = s["offsets"][i], counts[i]
        repetition, frequency, presence = penalties[i]
        for j in range(n):
            row = first + j
            mask = s["masks"][row] if s["words"] else (2 << j) - 1
            made = Counter(history[i][prompt:total])
            made.update(tokens[first + m] for m in range(n) if mask >> m & 1)
            every = sorted(set(history[i][:prompt]) | set(made))
            x = s["x"][row].to(F64)
            if every:
                at = torch.tensor(every, device="cuda")
                times = torch.tensor([made[t] for t in every], dtype=F64, device="cuda")
                y = x[at]
                y = torch.where(y > 0, y / repetition, y * repetition)
                x[at] = y - frequency * times - presence * (times > 0)
            mine = biases[begin[i]:begin[i + 1]]
            if mine:
                value = [struct.unpack("<f", struct.pack("<i", b))[0] for _, b in mine]
                x[torch.tensor([t for t, _ in mine], device="cuda")] += torch.tensor(
                    value, dtype=F64, device="cuda")
            if c["grammar"]:
                bits = (s["allowed"][row].long()[:, None] >> shift & 1).flatten()[:c["columns"]]
                x[bits == 0] = -math.inf
            out[row] = x
    return out


def _exact_keep(c, seed, s):
    pool = (c["layers"], s["pages"], 2, c["key_heads"], c["page_rows"], c["width"])
    cache, pr = _normal(seed, 1, pool, F16).to(F64), c["page_rows"]
    table = s["table"].tolist()
    for i, path in enumerate(_paths(c, seed, s["n"])):
        base = s["k"][i] - s["n"][i]
        for to, j in enumerate(path):
            p, r = base + to, base + j
            if to != j:
                cache[:, table[i][p // pr], :, :, p % pr] = cache[:, table[i][r // pr], :, :, r % pr]
    return cache


_EXACT = {"tables": _exact_tables, "slots": _exact_slots, "attention": _exact_attention,
          "logits": _exact_logits, "keep": _exact_keep}
