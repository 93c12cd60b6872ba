"""Steps with drafted trees as a program runs them: tables, maps, append, attention,
logits and the accepted rows' move, one after the other, against the whole text in
float64."""
from __future__ import annotations

import numpy as np
import pytest

from step_forms import adjust_logits, table_state, tree, words

HEADS, KEY_HEADS, WIDTH, VOCABULARY, PAGE_ROWS, COLUMNS, LAYERS = 4, 2, 64, 500, 8, 20, 2


class Model:
    """Two layers of attention between two embeddings, without positions: the tokens that
    a sequence has read decide, and where they stand does not."""

    def __init__(self, rng):
        d = HEADS * WIDTH
        self.embedding, self.output = (rng.standard_normal((VOCABULARY, d)).astype(np.float32) for _ in "io")
        self.k, self.v = (rng.standard_normal((LAYERS, d, KEY_HEADS * WIDTH)).astype(np.float32) * d ** -0.5 for _ in "kv")

    def layer(self, i, x):
        shape = (len(x), KEY_HEADS, WIDTH)
        return (x.astype(np.float16), (x @ self.k[i]).astype(np.float16).reshape(shape),
                (x @ self.v[i]).astype(np.float16).reshape(shape))

    def after(self, x, y):
        x = x + 2 * y.astype(np.float32).reshape(x.shape)
        return x / np.sqrt(np.mean(x * x, axis=1, keepdims=True))

    def logits(self, x):
        return (x @ self.output.T / 8).astype(np.float32)

    def embed(self, tokens):
        x = self.embedding[np.array(tokens)]
        return x / np.sqrt(np.mean(x * x, axis=1, keepdims=True))

    def whole(self, text, history, rounded=False):
        """Adjusted logits of every position of a text of one request in float64, of which
        the first `history` tokens count as a prompt; with `rounded`, with the fp16 values that
        pass between the operators."""
        x, n = self.embed(text).astype(np.float64), len(text)
        to = (lambda a: a.astype(np.float16).astype(np.float64)) if rounded else (lambda a: a)
        for i in range(LAYERS):
            q = to(x).reshape(n, HEADS, WIDTH)
            k, v = (to(x @ w[i].astype(np.float64)).reshape(n, KEY_HEADS, WIDTH) for w in (self.k, self.v))
            y = np.zeros((n, HEADS, WIDTH))
            for h in range(HEADS):
                score = q[:, h] @ k[:, h // 2].T * WIDTH ** -0.5
                p = np.where(np.tri(n, dtype=bool), np.exp(score - score.max(axis=1, keepdims=True)), 0.0)
                y[:, h] = to(to(p) @ v[:, h // 2] / to(p).sum(axis=1, keepdims=True))
            x = x + 2 * y.reshape(x.shape)
            x = x / np.sqrt(np.mean(x * x, axis=1, keepdims=True))
        raw, out = x @ self.output.T.astype(np.float64) / 8, []
        for i in range(n):  # the history of a position, and what came behind the prompt
            known = np.array([text[:i + 1]])
            out.append(adjust_logits(raw[i:i + 1], [0, 1], [VOCABULARY], None, known, [[min(history, i + 1), i + 1]], PENALTIES,
                                     [0, 0], ([], []), ALLOWED[None])[0][0])
        return np.array(out)


# What passes between the operators is rounded to fp16: that moves the logits of such a
# model by 0.005 (test_the_model_feels_no_rounding), whose best two are 0.6 apart on average.
# Twenty times that is allowed.
NEAR = 0.1
PENALTIES = np.array([[1.2, 0.3, 0.1]], np.float32)
ALLOWED = np.arange(VOCABULARY) % 32 != 3


def test_the_model_feels_no_rounding():
    """(CPU) What the roundings make of the logits, and how far apart the best two are."""
    rng = np.random.default_rng(30)
    model, gaps = Model(rng), []
    for n in (1, 20, 60):
        text = [int(t) for t in rng.integers(0, VOCABULARY, n)]
        exact = model.whole(text, 3)
        assert np.max(np.abs(model.whole(text, 3, rounded=True)[:, ALLOWED] - exact[:, ALLOWED])) <= NEAR / 5
        best = np.sort(exact, axis=1)[:, -2:]
        gaps += list(best[:, 1] - best[:, 0])
    assert np.mean(gaps) > 4 * NEAR


class Server:
    """Requests with their cache on the device; every step appends rows and gives the
    adjusted logits of all of them."""

    def __init__(self, ctx, model, pages, count):
        self.ctx, self.model, self.pages, self.count = ctx, model, pages, count
        rng = np.random.default_rng(5)
        free = [int(p) for p in rng.permutation(pages)]
        self.size = 2 + pages + count * (1 + COLUMNS)
        self.states = [ctx.upload(table_state(free, [[] for _ in range(count)], pages, COLUMNS)), ctx.alloc(4 * self.size)]
        shape = (LAYERS, pages, 2, KEY_HEADS, PAGE_ROWS, WIDTH)
        self.cache = ctx.upload(np.full(shape, np.nan, np.float16))
        self.layer_bytes = int(np.prod(shape[1:])) * 2
        self.lengths = np.zeros(count, np.int64)
        self.history = [[] for _ in range(count)]
        self.keep = []

    def up(self, a, dtype=np.int32):
        buf = self.ctx.upload(np.ascontiguousarray(np.array(a, dtype)))
        self.keep.append(buf)
        return buf

    def step(self, new, masks, source, prompt, first=False):
        """new: each sequence's tokens; masks of the rows; logits [rows, vocabulary].  first: they
        are prompts, whose tokens count as such (each sequence's last row is of use)."""
        ctx, m, count = self.ctx, self.model, self.count
        n = [len(t) for t in new]
        rows = sum(n)
        self.n, self.offsets_host = n, np.concatenate([[0], np.cumsum(n)])
        self.lengths = np.where(np.array(source) < 0, 0, self.lengths) + n
        wide = (max(n) + 31) // 32
        lengths, counts, mask = self.up(self.lengths), self.up(n), self.up(words(masks, wide), np.uint32)
        ctx.launch("ipu_stack_page_tables", self.states[1], [self.states[0], self.up(source), lengths],
                   [count, count, self.pages, PAGE_ROWS, COLUMNS])
        self.states.reverse()
        self.table = self.states[0].ptr + 4 * (2 + self.pages + count)
        maps = ctx.alloc(4 * (count + 1 + 2 * rows))
        self.keep.append(maps)
        ctx.launch("ipu_stack_slot_maps", maps, [counts, lengths, self.table, mask],
                   [count, rows, self.pages, PAGE_ROWS, COLUMNS, wide])
        self.length_buffer, self.offsets = lengths, maps.ptr
        self.positions = maps.download(np.int32)[count + 1:count + 1 + rows]
        tokens = np.concatenate([np.array(t, np.int32) for t in new])
        x = m.embed(tokens)
        freq = self.up([0.0], np.float32)
        out = self.ctx.alloc(rows * HEADS * WIDTH * 2)
        self.keep.append(out)
        for i in range(LAYERS):
            q, k, v = m.layer(i, x)
            cache = self.cache.ptr + i * self.layer_bytes
            ctx.launch("ipu_stack_append_pages_f16", cache,
                       [self.up(k, np.float16), self.up(v, np.float16), freq, self.table, self.offsets, lengths],
                       [count, rows, KEY_HEADS, WIDTH, KEY_HEADS * WIDTH, KEY_HEADS * WIDTH, 0, 0, 0, self.pages,
                        PAGE_ROWS, COLUMNS])
            ctx.launch("ipu_stack_attention_tree_pages_f16", out,
                       [self.up(q, np.float16), cache, self.table, self.offsets, lengths, mask],
                       [count, rows, max(n), HEADS, KEY_HEADS, WIDTH, HEADS * WIDTH, self.pages, PAGE_ROWS, COLUMNS, wide, 0])
            x = m.after(x, out.download(np.float16))
        if first:
            self.history = [list(t) for t in new]
        logits, result = self.up(m.logits(x), np.float32), ctx.alloc(rows * VOCABULARY * 4)
        self.keep.append(result)
        width = max(1, max(len(h) for h in self.history))
        history = np.zeros((count, width), np.int32)
        for s, h in enumerate(self.history):
            history[s, :len(h)] = h
        allowed = np.full((rows, (VOCABULARY + 31) // 32), 0xfffffff7, np.uint32)  # of each word, token 3 is not
        ctx.launch("ipu_stack_adjust_logits_f32", result,
                   [logits, self.offsets, self.up(tokens * 0 - 1 if first else tokens), mask, self.up(history),
                    self.up([[min(prompt[s], len(h)), len(h)] for s, h in enumerate(self.history)]),
                    self.up(np.repeat(PENALTIES, count, axis=0), np.float32), self.up([0] * (count + 1)), self.up([0, 0]),
                    self.up(allowed, np.uint32)],
                   [count, rows, VOCABULARY, VOCABULARY, VOCABULARY, wide, width, 0, allowed.shape[1]])
        return result.download(np.float32).reshape(rows, VOCABULARY)

    def accept(self, paths):
        """Rows of each sequence that stay."""
        width = max(1, max(len(p) for p in paths))
        path = [p + [-1] * (width - len(p)) for p in paths]
        self.ctx.launch("ipu_stack_keep_pages_f16", self.cache,
                        [self.table, self.offsets, self.length_buffer, self.up(path), self.up([len(p) for p in paths])],
                        [self.count, sum(self.n), LAYERS, KEY_HEADS, WIDTH, self.pages, PAGE_ROWS, COLUMNS, width])
        self.lengths = self.lengths - self.n + [len(p) for p in paths]

    def close(self):
        self.ctx.sync()
        for b in self.keep + self.states + [self.cache]:
            b.free()


def chain(n):
    return [(2 << i) - 1 for i in range(n)]


def run(ctx, model, prompts, steps, drafts, rng, known):
    """Greedy tokens of each request, `drafts` rows verified at once, some of them of the
    texts that are `known`; and how many were accepted."""
    count = len(prompts)
    server = Server(ctx, model, 150, count)
    prompt = [len(p) for p in prompts]
    logits = server.step(prompts, [m for p in prompts for m in chain(len(p))], [-1] * count, prompt, True)
    produced = [[int(np.argmax(logits[int(server.offsets_host[s + 1]) - 1]))] for s in range(count)]
    accepted = 0
    while min(len(p) for p in produced) < steps:
        new, masks, trees = [], [], []
        for s in range(count):
            mine = tree(rng, drafts)
            tokens = [produced[s][-1]] + [int(t) for t in rng.integers(0, VOCABULARY, drafts - 1)]
            for j in range(1, drafts):
                at = len(produced[s]) - 1 + bin(mine[j]).count("1") - 1
                if at < len(known[s]) and rng.random() < 0.8:
                    tokens[j] = known[s][at]
            new.append(tokens)
            masks += mine
            trees.append(mine)
        logits = server.step(new, masks, list(range(count)), prompt)
        assert np.array_equal(server.positions, np.concatenate(
            [[server.lengths[s] - drafts + bin(m).count("1") - 1 for m in trees[s]] for s in range(count)]))
        paths = []
        for s in range(count):
            first, path, node = int(server.offsets_host[s]), [0], 0
            while True:
                best = int(np.argmax(logits[first + node]))
                produced[s].append(best)
                child = [j for j in range(node + 1, drafts)
                         if trees[s][j] == trees[s][node] | 1 << j and new[s][j] == best]
                if not child:
                    break
                node = child[0]
                path.append(node)
            accepted += len(path) - 1
            server.history[s] += [new[s][j] for j in path]
            paths.append(path)
        server.accept(paths)
    server.close()
    return produced, accepted


@pytest.mark.gpu
def test_drafted_tokens_change_nothing(ctx):
    """Tokens taken one at a time, and verified by trees of 7 and 25 drafts of which many are
    right: each is the best of the whole text before it."""
    rng = np.random.default_rng(31)
    model = Model(rng)
    prompts = [[int(t) for t in rng.integers(0, VOCABULARY, n)] for n in (5, 1, 19)]
    known = [[] for _ in prompts]
    for drafts in (1, 7, 25):
        got, accepted = run(ctx, model, prompts, 24, drafts, rng, known)
        assert accepted == 0 if drafts == 1 else accepted > 20
        if drafts == 1:
            known = got
        for p, text in zip(prompts, got):
            logits = model.whole(p + text, len(p))
            for i, token in enumerate(text):
                assert logits[len(p) - 1 + i].max() - logits[len(p) - 1 + i][token] <= 2 * NEAR, (drafts, i)


@pytest.mark.gpu
def test_requests_end_and_begin(ctx):
    """A request that ends gives its pages to the next one, which reads nothing of it."""
    rng = np.random.default_rng(32)
    model = Model(rng)
    texts = [[int(t) for t in rng.integers(0, VOCABULARY, n)] for n in (60, 45, 30, 50)]
    server = Server(ctx, model, 16, 2)  # 128 positions: two texts fit, three do not
    for pair in [(0, 1), (2, 3), (1, 0), (3, 2)]:
        new = [texts[t] for t in pair]
        logits = server.step(new, [m for t in new for m in chain(len(t))], [-1, -1], [len(t) for t in new], True)
        for s, t in enumerate(pair):
            got, want = logits[server.offsets_host[s + 1] - 1], model.whole(texts[t], len(texts[t]))[-1]
            assert np.array_equal(np.isfinite(got), ALLOWED) and np.all(np.abs(got - want)[ALLOWED] <= NEAR)
        state = server.states[0].download(np.int32)
        assert state[1] == 0 and state[0] == 16 - sum(-(-len(t) // PAGE_ROWS) for t in new)
    server.close()
