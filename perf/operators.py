"""The decoder's serving operators as programs run them on one MI355X: rotary
positions, norms of query and key heads with the rotation, appends to a paged
cache of keys and values, and attention of a ragged batch over that cache,
also with a prefix that the whole batch shares.

Each case is a dict of plain values; `prepare` makes its inputs on the GPU and
what a program keeps between calls, `run` is one pass: through the kernel ABI
where `own` is true, in elementary torch operations in 32 bits where it is
false.  `exact` is the operator's definition in 64 bits.

The cache is [pages][2][key heads][page rows][width] fp16, keys before values;
row p of sequence s lies in page table[s][p / page_rows] at row p % page_rows.
A batch is ragged: rows offsets[s] .. offsets[s + 1] - 1 belong to sequence s,
the last of them at position lengths[s] - 1.
"""
import math
import random
import struct

import torch

own = False

F16, F32, F64 = torch.float16, torch.float32, torch.float64

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
def rotary(rows, heads, width, rotary_width, interleaved, f32, scaling, first):
    """Positions first .. first + rows - 1 on rows of `heads` heads; `scaling`
    is how the frequencies reach past the trained context."""
    return {"kind": "rotary", "rows": rows, "heads": heads, "width": width,
            "rotary_width": rotary_width, "interleaved": interleaved, "f32": f32,
            "scaling": scaling, "first": first}


def norm_rotary(rows, query_heads, key_heads, width, rotary_width, interleaved, f32, first):
    """Query and key heads of the rows of a fused projection [rows, query +
    2 key heads, width]; the value heads stay behind."""
    return {"kind": "norm_rotary", "rows": rows, "query_heads": query_heads,
            "key_heads": key_heads, "width": width, "rotary_width": rotary_width,
            "interleaved": interleaved, "f32": f32, "first": first}


def append(sequences, rows, keys, key_heads, width, rotary_width, interleaved, page_rows,
           pattern, padding):
    """Up to `rows` new tokens of each sequence, whose length after them is up
    to `keys`; `padding` rows behind the last sequence."""
    return {"kind": "append", "sequences": sequences, "rows": rows, "keys": keys,
            "key_heads": key_heads, "width": width, "rotary_width": rotary_width,
            "interleaved": interleaved, "page_rows": page_rows, "pattern": pattern,
            "padding": padding}


def attention(sequences, rows, keys, shared, query_heads, key_heads, width, page_rows, causal,
              batch, pattern, padding):
    """`batch` says what the sequences are: "equal" (rows and keys each),
    "ragged" (1 .. rows new tokens, keys / 16 .. keys in all, spread over
    their logarithm) or "mixed" (one chunk of `rows`, single tokens else)."""
    return {"kind": "shared" if shared else "attention", "sequences": sequences, "rows": rows,
            "keys": keys, "shared": shared, "query_heads": query_heads, "key_heads": key_heads,
            "width": width, "page_rows": page_rows, "causal": causal, "batch": batch,
            "pattern": pattern, "padding": padding}


def listed():
    return [
        # One step of a decoding batch: 16 heads of 128, where the launch is
        # everything.
        dict(rotary(64, 16, 128, 128, False, False, "none", 4000), name="rotary_decode"),
        # A long prompt's queries in fp32, half of each head rotated, far past
        # the trained context (frequencies scaled by their wavelength).
        dict(rotary(16384, 16, 128, 64, True, True, "banded", 1000000), name="rotary_long"),
        # One step: query and key heads of 8 tokens' fused projections.
        dict(norm_rotary(8, 32, 8, 128, 128, False, False, 511), name="norm_rotary_decode"),
        # Prefill: the same for a prompt batch of 16384 tokens.
        dict(norm_rotary(16384, 32, 8, 128, 128, False, False, 0), name="norm_rotary_prefill"),
        # One step of 64 sequences into pages of 16 rows.
        dict(append(64, 1, 4096, 8, 128, 128, False, 16, 1, 0), name="append_decode"),
        # Prompts of odd lengths, padded at the end, into pages of 64 rows.
        dict(append(16, 2000, 4096, 8, 128, 128, False, 64, 2, 37), name="append_prefill"),
        # The smallest step: 4 sequences of up to 1024 tokens.
        dict(attention(4, 1, 1024, 0, 16, 16, 64, 16, True, "ragged", 3, 0),
             name="attention_decode_small"),
        # A serving step: 64 sequences of very different lengths.
        dict(attention(64, 1, 32768, 0, 32, 8, 128, 64, True, "ragged", 4, 0),
             name="attention_decode_ragged"),
        # Chunks of prompts against what the cache already holds.
        dict(attention(4, 2048, 8192, 0, 32, 8, 128, 64, True, "equal", 5, 0),
             name="attention_chunks"),
        # One prompt's chunk beside decoding sequences, odd widths, padded.
        dict(attention(17, 333, 3001, 0, 16, 16, 72, 32, True, "mixed", 6, 5),
             name="attention_mixed_odd"),
        # A small batch behind one system prompt.
        dict(attention(8, 1, 2100, 2048, 16, 4, 128, 16, True, "equal", 7, 0),
             name="shared_small"),
        # Many sequences behind a long shared document.
        dict(attention(128, 1, 17000, 16384, 32, 8, 128, 64, True, "equal", 8, 0),
             name="shared_long"),
    ]


def _log_size(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the same ranges: a kind, then sizes over its range."""
    kind = rng.choice(["rotary", "norm_rotary", "append", "attention", "attention", "chunk",
                       "shared"])
    width = rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 128, 192, 256])
    part = rng.choice([width, width, width // 2 // 2 * 2, width // 4 // 2 * 2])
    interleaved = rng.random() < 0.5
    if kind == "rotary":
        while True:
            rows, heads = _log_size(rng, 1, 16384), rng.choice([1, 2, 8, 12, 16, 32])
            if rows * heads * width <= 16384 * 16 * 128:
                break
        return rotary(rows, heads, width, part, interleaved, rng.random() < 0.4,
                      rng.choice(["none", "linear", "base", "banded"]), _log_size(rng, 1, 1 << 20))
    if kind == "norm_rotary":
        while True:
            rows = _log_size(rng, 1, 16384)
            heads, keys = rng.choice([(12, 12), (16, 16), (16, 4), (32, 8), (32, 1), (5, 0)])
            if rows * (heads + keys) * width <= 16384 * 40 * 128:
                break
        return norm_rotary(rows, heads, keys, width, part, interleaved, rng.random() < 0.4,
                           _log_size(rng, 1, 1 << 20))
    page_rows = rng.choice([8, 16, 16, 32, 64, 128])
    pattern, padding = rng.randrange(1 << 20), rng.choice([0, 0, rng.randint(1, 100)])
    key_heads, group = rng.choice([(16, 1), (12, 1), (8, 4), (8, 8), (4, 4), (2, 7), (1, 16)])
    if kind == "append":
        while True:
            sequences, rows = _log_size(rng, 1, 256), _log_size(rng, 1, 4096)
            keys = max(rows, _log_size(rng, 1, 8192))
            if (sequences * rows * key_heads * width <= 16 * 2000 * 8 * 128
                    and sequences * keys * key_heads * width <= 64 * 4096 * 8 * 128):
                break
        return append(sequences, rows, keys, key_heads, width, rng.choice([0, part]), interleaved,
                      page_rows, pattern, padding)
    if kind == "attention":
        # Single tokens and the few of a draft's verification.
        while True:
            sequences, keys = _log_size(rng, 1, 256), _log_size(rng, 1, 65536)
            if sequences * keys * key_heads * width <= 64 * 16384 * 8 * 128:
                break
        return attention(sequences, rng.choice([1, 1, 1, 1, 2, 5]), keys, 0, key_heads * group,
                         key_heads, width, page_rows, rng.random() < 0.8,
                         rng.choice(["equal", "ragged", "ragged"]), pattern, padding)
    if kind == "chunk":
        while True:
            sequences, rows = _log_size(rng, 1, 32), _log_size(rng, 16, 4096)
            keys = max(rows, _log_size(rng, 16, 16384))
            if (sequences * rows * keys * key_heads * group * width <= 2048 * 8192 * 32 * 128 * 2
                    and sequences * keys * key_heads * width <= 64 * 16384 * 8 * 128):
                break
        return attention(sequences, rows, keys, 0, key_heads * group, key_heads, width, page_rows,
                         rng.random() < 0.8, rng.choice(["equal", "ragged", "mixed"]), pattern,
                         padding)
    while True:
        sequences, shared = _log_size(rng, 2, 256), _log_size(rng, 64, 32768)
        own_keys = _log_size(rng, 1, 2048)
        if (sequences * own_keys * key_heads * width <= 128 * 616 * 8 * 128
                and sequences * shared * key_heads * group * width <= 128 * 16384 * 32 * 128):
            break
    return attention(sequences, rng.choice([1, 1, 1, 3]), shared + own_keys, shared,
                     key_heads * group, key_heads, width, page_rows, True,
                     rng.choice(["equal", "ragged"]), pattern, padding)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(seed, tensor, shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 16 + tensor)
    return torch.randn(shape, generator=g, device="cuda", dtype=F32).mul_(scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _frequencies(c):
    """fp32 [rotary_width / 2] and the factor on the rotated elements: base^(-2 i
    / r), and its forms for a context 8 times the trained 4096."""
    r, base, factor, trained = c["rotary_width"], 10000.0, 8.0, 4096.0
    scaling = c.get("scaling", "none")
    if scaling == "base":
        base *= factor ** (r / max(r - 2.0, 1.0))
    f = base ** (-torch.arange(r // 2, dtype=F64) * 2.0 / max(r, 1))
    if scaling == "linear":
        f = f / factor
    elif scaling == "banded":
        turns = trained * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
    magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "banded" else 1.0
    # At least one element, so that there is an array to pass.
    f = f.to(F32) if r else torch.zeros(1, dtype=F32)
    return f.to("cuda"), struct.unpack("<f", struct.pack("<f", magnitude))[0]


def _batch(c):
    """Rows and lengths of the sequences, of the case alone."""
    rng = random.Random(c["pattern"])
    n, k = [], []
    for s in range(c["sequences"]):
        if c["kind"] == "append":
            rows = rng.randint(max(1, c["rows"] // 2), c["rows"])
            n.append(rows)
            k.append(rng.randint(rows, c["keys"]))
            continue
        least = c["shared"] + 1 if c["shared"] else 1
        if c["batch"] == "equal":
            rows, keys = c["rows"], c["keys"]
        elif c["batch"] == "ragged":
            rows = rng.randint(1, c["rows"])
            low = max(least, c["keys"] // 16)
            keys = _log_size(rng, low, max(low, c["keys"]))
        else:
            rows = c["rows"] if s == c["sequences"] // 2 else 1
            keys = rng.randint(max(least, c["keys"] // 2), c["keys"])
        k.append(keys)
        # New tokens are among the keys they see.
        n.append(min(rows, max(1, keys - c["shared"])))
    return n, k


def _cache(c, seed):
    """Cache, table and the batch's arrays: pages handed out in no order, a
    few free ones, table entries past a sequence's end -1."""
    n, k = _batch(c)
    pr, shared = c["page_rows"], c.get("shared", 0)
    rng = random.Random(c["pattern"] * 1000003 + seed)
    need = [(x + pr - 1) // pr for x in k]
    columns = max(need) + 2
    common = shared // pr  # pages that every sequence shares whole
    pages = sum(need) - common * (len(k) - 1) + 3
    free = list(range(pages))
    rng.shuffle(free)
    prefix = [free.pop() for _ in range(common)]
    table = []
    for x in need:
        mine = prefix + [free.pop() for _ in range(x - common)]
        table.append(mine + [-1] * (columns - x))
    cache = _normal(seed, 1, (pages, 2, c["key_heads"], pr, c["width"]), F16)
    offsets = [0]
    for x in n:
        offsets.append(offsets[-1] + x)
    if shared % pr:
        # The page in which the prefix ends: a copy of its first rows in each.
        first = cache[table[0][common]]
        others = torch.tensor([t[common] for t in table[1:]], device="cuda")
        cache[others, :, :, :shared % pr] = first[:, :, :shared % pr]
    return {"n": n, "k": k, "cache": cache, "columns": columns, "pages": pages,
            "offsets": offsets, "rows": offsets[-1] + c["padding"], "table": _ints(table),
            "row_offsets": _ints(offsets), "lengths": _ints(k)}


def prepare(case, seed):
    c = case
    state = {"case": c}
    if c["kind"] in ("rotary", "norm_rotary"):
        dtype, rows, width = F32 if c["f32"] else F16, c["rows"], c["width"]
        heads = c["heads"] if c["kind"] == "rotary" else c["query_heads"] + c["key_heads"]
        extra = 0 if c["kind"] == "rotary" else c["key_heads"]
        state["x"] = _normal(seed, 1, (rows, heads + extra, width), dtype)
        state["out"] = torch.empty((rows, heads, width), dtype=dtype, device="cuda")
        state["positions"] = _ints([c["first"] + i for i in range(rows)])
        state["frequencies"], state["magnitude"] = _frequencies(c)
        if c["kind"] == "norm_rotary":
            state["weights"] = [_normal(seed, t, (width,), F32, 0.1).add_(1.0).to(dtype)
                                for t in (2, 3)]
    else:
        state.update(_cache(c, seed))
        rows, width = state["rows"], c["width"]
        if c["kind"] == "append":
            state["keys"] = _normal(seed, 2, (rows, c["key_heads"], width), F16)
            state["values"] = _normal(seed, 3, (rows, c["key_heads"], width), F16)
            state["frequencies"], state["magnitude"] = _frequencies(c)
            # Where the plain form writes: the page and row of each new token.
            table, where = state["table"].tolist(), []
            for s, (n, k) in enumerate(zip(state["n"], state["k"])):
                where += [(table[s][p // c["page_rows"]], p % c["page_rows"], p)
                          for p in range(k - n, k)]
            where = torch.tensor(where, device="cuda")
            state["page"], state["row"], state["positions"] = where.unbind(1)
        else:
            state["q"] = _normal(seed, 2, (rows, c["query_heads"], width), F16, 1.5)
            state["out"] = torch.zeros((rows, c["query_heads"], width), dtype=F16, device="cuda")
    # What a program keeps for its launches: the addresses and sizes.
    state["call"] = _call(state)
    # The inputs were made on torch's stream, the library has its own.
    torch.cuda.synchronize()
    return state


def _bits(x):
    return struct.unpack("<I", struct.pack("<f", x))[0]


def _call(state):
    """Symbol, output, inputs and scalars of the case's launch."""
    c, s = state["case"], state
    width = c["width"]
    if c["kind"] == "rotary":
        h = c["heads"]
        return ("ipu_stack_rotary_f32" if c["f32"] else "ipu_stack_rotary_f16", s["out"].data_ptr(),
                [t.data_ptr() for t in (s["x"], s["positions"], s["frequencies"])],
                [c["rows"], h, width, c["rotary_width"], int(c["interleaved"]), h * width, width,
                 h * width, width, _bits(s["magnitude"])])
    if c["kind"] == "norm_rotary":
        h, k = c["query_heads"], c["key_heads"]
        return ("ipu_stack_norm_rotary_f32" if c["f32"] else "ipu_stack_norm_rotary_f16",
                s["out"].data_ptr(),
                [t.data_ptr() for t in (s["x"], *s["weights"], s["positions"], s["frequencies"])],
                [c["rows"], h, k, width, c["rotary_width"], int(c["interleaved"]),
                 (h + 2 * k) * width, (h + k) * width, _bits(1e-6), _bits(s["magnitude"])])
    if c["kind"] == "append":
        pitch = c["key_heads"] * width
        return ("ipu_stack_append_pages_f16", s["cache"].data_ptr(),
                [t.data_ptr() for t in (s["keys"], s["values"], s["frequencies"], s["table"],
                                        s["row_offsets"], s["lengths"])],
                [c["sequences"], s["rows"], c["key_heads"], width, pitch, pitch, c["rotary_width"],
                 int(c["interleaved"]), _bits(s["magnitude"]), s["pages"], c["page_rows"],
                 s["columns"]])
    scalars = [c["sequences"], s["rows"], max(s["n"]), c["query_heads"], c["key_heads"], width,
               c["query_heads"] * width, s["pages"], c["page_rows"], s["columns"],
               int(c["causal"]), 0]
    symbol = "ipu_stack_attention_pages_f16"
    if c["kind"] == "shared":
        symbol = "ipu_stack_attention_shared_pages_f16"
        scalars.append(c["shared"])
    return (symbol, s["out"].data_ptr(),
            [t.data_ptr() for t in (s["q"], s["cache"], s["table"], s["row_offsets"],
                                    s["lengths"])], scalars)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        _context().launch(*state["call"])
        return state["cache"] if state["case"]["kind"] == "append" else state["out"]
    return _PLAIN[state["case"]["kind"]](state)


def _rotate(x, positions, frequencies, magnitude, rotary_width, interleaved):
    """fp32 [rows, heads, width]; the angles in 64 bits."""
    if rotary_width == 0:
        return x
    angles = positions.to(F64)[:, None] * frequencies.to(F64)[None, :]
    cos = (torch.cos(angles) * magnitude).to(F32)[:, None, :]
    sin = (torch.sin(angles) * magnitude).to(F32)[:, None, :]
    turned, rest = x[..., :rotary_width], x[..., rotary_width:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :rotary_width // 2], turned[..., rotary_width // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_rotary(s):
    c = s["case"]
    y = _rotate(s["x"].to(F32), s["positions"], s["frequencies"], s["magnitude"],
                c["rotary_width"], c["interleaved"])
    return s["out"].copy_(y)


def _plain_norm_rotary(s):
    c = s["case"]
    q, k = c["query_heads"], c["key_heads"]
    x = s["x"][:, :q + k].to(F32)
    w = torch.cat([t.to(F32)[None].expand(n, -1) for t, n in zip(s["weights"], (q, k))])
    y = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6) * w
    return s["out"].copy_(_rotate(y, s["positions"], s["frequencies"], s["magnitude"],
                                  c["rotary_width"], c["interleaved"]))


def _plain_append(s):
    c = s["case"]
    rows = s["offsets"][-1]
    keys = _rotate(s["keys"][:rows].to(F32), s["positions"], s["frequencies"], s["magnitude"],
                   c["rotary_width"], c["interleaved"])
    s["cache"][s["page"], 0, :, s["row"]] = keys.to(F16)
    s["cache"][s["page"], 1, :, s["row"]] = s["values"][:rows]
    return s["cache"]


def _plain_attention(s):
    c = s["case"]
    heads, width, scale = c["key_heads"], c["width"], c["width"] ** -0.5
    group = c["query_heads"] // heads
    for i, (n, k) in enumerate(zip(s["n"], s["k"])):
        used = (k + c["page_rows"] - 1) // c["page_rows"]
        pages = s["cache"][s["table"][i, :used].long()]
        # [pages, 2, heads, rows, width] -> [2, heads, keys, width]
        kv = pages.permute(1, 2, 0, 3, 4).reshape(2, heads, -1, width)[:, :, :k].to(F32)
        start = s["offsets"][i]
        q = s["q"][start:start + n].to(F32).reshape(n, heads, group, width).transpose(0, 1)
        x = torch.matmul(q.reshape(heads, n * group, width), kv[0].transpose(1, 2).contiguous())
        x = x.mul_(scale).reshape(heads, n, group, k)
        if c["causal"] and n > 1:
            # The first row sees the keys up to k - n, the last all.
            late = (torch.arange(k, device="cuda")[None, :]
                    > torch.arange(k - n, k, device="cuda")[:, None])
            x = x.masked_fill_(late[None, :, None], -math.inf)
        p = x.sub_(x.amax(dim=3, keepdim=True)).exp_()
        y = torch.matmul(p.reshape(heads, n * group, k), kv[1])
        y = y.reshape(heads, n, group, width) / p.sum(dim=3, keepdim=True)
        s["out"][start:start + n] = y.transpose(0, 1).reshape(n, heads * group, width)
    return s["out"]


_PLAIN = {"rotary": _plain_rotary, "norm_rotary": _plain_norm_rotary, "append": _plain_append,
          "attention": _plain_attention, "shared": _plain_attention}


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its exact result
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] in ("rotary", "norm_rotary"):
        heads = c["heads"] if c["kind"] == "rotary" else c["query_heads"] + c["key_heads"]
        elements, size = c["rows"] * heads * c["width"], 4 if c["f32"] else 2
        pairs = c["rows"] * heads * c["rotary_width"] // 2
        extra = 2 * c["width"] * size if c["kind"] == "norm_rotary" else 0
        return {"bytes": 2 * elements * size + 4 * c["rows"] + 2 * c["rotary_width"] + extra,
                "flops": 6 * pairs + (4 * elements if extra else 0)}
    n, k = _batch(c)
    if c["kind"] == "append":
        elements = sum(n) * c["key_heads"] * c["width"]
        return {"bytes": 8 * elements + 4 * (3 * len(n) + sum(n)),
                "flops": 3 * sum(n) * c["key_heads"] * c["rotary_width"]}
    shared = c["shared"]
    keys = shared + sum(x - shared for x in k)
    moved = 2 * 2 * keys * c["key_heads"] * c["width"]
    moved += 2 * 2 * sum(n) * c["query_heads"] * c["width"]
    table = sum((x + c["page_rows"] - 1) // c["page_rows"] for x in k)
    pairs = sum(a * b - (a * (a - 1) // 2 if c["causal"] else 0) for a, b in zip(n, k))
    return {"bytes": moved + 4 * (2 * len(n) + 1 + table),
            "flops": 4 * pairs * c["query_heads"] * c["width"]}


def _exact_rotation(x, first_positions, f, magnitude, r, interleaved):
    """In place on float64 [rows, heads, width], as a complex product."""
    if r:
        turn = torch.polar(torch.full((1,), magnitude, dtype=F64, device="cuda"),
                           first_positions.to(F64)[:, None] * f.to(F64)[None, :])[:, None]
        index = torch.arange(r // 2, device="cuda")
        a, b = (2 * index, 2 * index + 1) if interleaved else (index, index + r // 2)
        z = torch.complex(x[..., a], x[..., b]) * turn
        x[..., a], x[..., b] = z.real, z.imag
    return x


def exact(case, seed):
    c = case
    if c["kind"] in ("rotary", "norm_rotary"):
        f, magnitude = _frequencies(c)
        dtype, rows, width = F32 if c["f32"] else F16, c["rows"], c["width"]
        if c["kind"] == "rotary":
            x = _normal(seed, 1, (rows, c["heads"], width), dtype).to(F64)
        else:
            q, k = c["query_heads"], c["key_heads"]
            x = _normal(seed, 1, (rows, q + 2 * k, width), dtype)[:, :q + k].to(F64)
            x = x / torch.sqrt((x ** 2).sum(dim=-1, keepdim=True) / width + 1e-6)
            for t, part in ((2, slice(0, q)), (3, slice(q, q + k))):
                x[:, part] *= _normal(seed, t, (width,), F32, 0.1).add_(1.0).to(dtype).to(F64)
        positions = torch.arange(c["first"], c["first"] + rows, device="cuda")
        return _exact_rotation(x, positions, f, magnitude, c["rotary_width"], c["interleaved"])
    batch = _cache(c, seed)
    table, pr = batch["table"].tolist(), c["page_rows"]
    if c["kind"] == "append":
        f, magnitude = _frequencies(c)
        rows = batch["rows"]
        keys, values = (_normal(seed, t, (rows, c["key_heads"], c["width"]), F16).to(F64)
                        for t in (2, 3))
        out = batch["cache"].to(F64)
        start = 0
        for s, (n, k) in enumerate(zip(batch["n"], batch["k"])):
            positions = torch.arange(k - n, k, device="cuda")
            page = batch["table"][s].long()[positions // pr]
            turned = _exact_rotation(keys[start:start + n], positions, f, magnitude,
                                     c["rotary_width"], c["interleaved"])
            out[page, 0, :, positions % pr] = turned
            out[page, 1, :, positions % pr] = values[start:start + n]
            start += n
        return out
    if work(c)["flops"] > 2.5e12:  # too long in 64 bits
        return None
    queries = _normal(seed, 2, (batch["rows"], c["query_heads"], c["width"]), F16, 1.5)
    out = torch.zeros(queries.shape, dtype=F64, device="cuda")
    group = c["query_heads"] // c["key_heads"]
    start = 0
    for s, (n, k) in enumerate(zip(batch["n"], batch["k"])):
        place = torch.arange(k, device="cuda")
        page, row = batch["table"][s].long()[place // pr], place % pr
        for h in range(c["query_heads"]):
            key = batch["cache"][page, 0, h // group, row].to(F64)
            value = batch["cache"][page, 1, h // group, row].to(F64)
            x = torch.mm(queries[start:start + n, h].to(F64), key.t().contiguous())
            x = x / math.sqrt(c["width"])
            if c["causal"]:
                position = place[k - n:][:, None]
                x = torch.where(place[None, :] <= position, x, -math.inf)
            out[start:start + n, h] = torch.mm(torch.softmax(x, dim=1), value)
        start += n
    return out
