"""The cache in pages on the GPU: its writes against the device's other RoPE's
bits, its attention against a plain form in 64 bits (tolerances derived in
paged_reference.attention), and both with the sampler as a server runs them."""
import numpy as np
import pytest

import paged_reference as ref
import tensomite_hip as th

pytestmark = pytest.mark.gpu

HEADS = [(9, 3, 64), (4, 4, 64), (8, 1, 128), (6, 2, 80), (4, 2, 8), (2, 1, 256)]


def say(*args):
    print(*args, flush=True)


@pytest.fixture(scope="module")
def dev():
    return th.HIPDevice(0)


def cache_of(dev, kind, batch, kv, keys, values):
    raw_k, k = ref.to_kind(keys, kind)
    raw_v, v = ref.to_kind(values, kind)
    cache = dev.paged_cache(kind, batch.pages, batch.page_size, kv, keys.shape[-1], keys=dev.from_array(raw_k),
                            values=dev.from_array(raw_v))
    return cache, k, v


def inputs(seed, batch, heads, kv, width):
    rng = np.random.default_rng(seed)
    shape = (batch.pages, kv, batch.page_size, width)
    q = rng.normal(0, 1.5, (batch.tokens, heads, width)).astype(np.float32)
    if batch.tokens:
        q[batch.tokens // 2] *= 8.0  # a sharp softmax
    return q, rng.normal(0, 1, shape).astype(np.float32), rng.normal(0, 1, shape).astype(np.float32)


def attend(dev, kind, batch, q, keys, values, window=0, sinks=0, scale=None):
    tokens, heads, width = q.shape
    scale = float(np.float32(1.0 / np.sqrt(width))) if scale is None else scale
    cache, k, v = cache_of(dev, kind, batch, keys.shape[1], keys, values)
    fill = np.full((tokens, heads, width), 7.25, np.float32)
    dst = dev.from_array(fill)
    dev.attention_paged(dev.from_array(q), tokens, heads, cache, batch.on(dev), scale, window=window, sinks=sinks,
                        dst=dst)
    got = dev.to_array(dst, np.float32, q.size).reshape(q.shape)
    dev.sync()
    want, tol = ref.attention(q, k, v, batch, scale, window, sinks)
    return got, want, tol


def agree(got, want, tol, batch):
    mine = np.zeros(got.shape[0], bool)
    mine[batch.starts[0]:batch.starts[-1]] = True
    assert (got[~mine] == 7.25).all()  # rows of no sequence are left as they were
    error = np.abs(got[mine] - want[mine]).max(-1)
    worst = float((error / tol[mine]).max()) if error.size else 0.0
    say("error of the tolerance", worst)
    assert not np.isnan(got[mine]).any()
    assert worst <= 1.0


BATCHES = {
    "one token": [(1, 1)],
    "one step": [(1, 77)],
    "steps": [(1, 1), (1, 300), (1, 64), (1, 65), (1, 513)],
    "no tokens between": [(0, 40), (1, 33), (0, 0), (2, 2), (0, 9)],
    "few": [(3, 50), (5, 5), (2, 190), (4, 64)],
    "prompt": [(97, 97)],
    "chunks": [(70, 200), (1, 130), (33, 33), (150, 151)],
}


@pytest.mark.parametrize("kind", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("name", list(BATCHES))
@pytest.mark.parametrize("heads,kv,width", HEADS[:2])
def test_attention_of_batches(dev, kind, name, heads, kv, width):
    say("batch", kind, name, heads, kv, width)
    batch = ref.Batch(BATCHES[name], 16, seed=3, lead=2, trail=3)
    q, keys, values = inputs(5, batch, heads, kv, width)
    agree(*attend(dev, kind, batch, q, keys, values), batch)


@pytest.mark.parametrize("kind", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("heads,kv,width", HEADS[2:])
@pytest.mark.parametrize("page_size", [1, 24, 128])
def test_attention_of_shapes(dev, kind, heads, kv, width, page_size):
    say("shape", kind, heads, kv, width, page_size)
    batch = ref.Batch([(1, 90), (40, 140), (2, 35)], page_size, seed=4)
    q, keys, values = inputs(6, batch, heads, kv, width)
    agree(*attend(dev, kind, batch, q, keys, values), batch)


@pytest.mark.parametrize("kind", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (64, 0), (63, 70), (100, 1), (5000, 3), (37, 600)])
def test_attention_with_a_window(dev, kind, window, sinks):
    say("window", kind, window, sinks)
    batch = ref.Batch([(1, 500), (80, 300), (3, 70), (1, 1), (20, 20)], 32, seed=5)
    q, keys, values = inputs(7, batch, 6, 3, 64)
    agree(*attend(dev, kind, batch, q, keys, values, window, sinks), batch)


@pytest.mark.parametrize("kind", ["F32", "F16"])
@pytest.mark.parametrize("heads,kv,width", [(8, 8, 64), (8, 2, 128)])
def test_attention_of_long_sequences(dev, kind, heads, kv, width):
    # split over the positions and joined; lengths that leave splits empty
    say("long", kind, heads, kv, width)
    batch = ref.Batch([(1, 9000), (1, 3), (2, 4097), (20, 2500)], 64, seed=6)
    q, keys, values = inputs(8, batch, heads, kv, width)
    agree(*attend(dev, kind, batch, q, keys, values), batch)
    agree(*attend(dev, kind, batch, q, keys, values, window=3000, sinks=2), batch)


@pytest.mark.parametrize("kind", ["F32", "F16", "BF16"])
def test_scores_of_any_size(dev, kind):
    # large and tiny queries and keys, a scale of nothing, a negative one
    batch = ref.Batch([(1, 200), (50, 120)], 16, seed=7)
    for seed, (fq, fk, scale) in enumerate([(60.0, 1.0, 0.125), (1e-4, 200.0, 0.125), (1e4, 1e-3, 0.3), (1.0, 1.0, 0.0),
                                            (2.0, 1.0, -0.2)]):
        say("scores", kind, fq, fk, scale)
        q, keys, values = inputs(20 + seed, batch, 4, 2, 64)
        agree(*attend(dev, kind, batch, q * np.float32(fq), keys * np.float32(fk), values, scale=scale), batch)


@pytest.mark.parametrize("kind", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_hidden_positions_do_not_reach_a_result(dev, kind, bad):
    # every place no token sees holds `bad`, and a later token's key and value do too
    say("hidden", kind, bad)
    window, sinks = 20, 3
    batch = ref.Batch([(1, 100), (30, 90), (70, 70)], 16, seed=8)
    q, keys, values = inputs(9, batch, 4, 2, 64)
    hold = np.ones(keys.shape, bool)
    for s, (c, n) in enumerate(zip(batch.new, batch.lengths)):
        page, place = batch.slots(s)
        seen = np.zeros(n, bool)
        for i in range(c):
            seen |= ref.visible(n - c + i, np.arange(n), window, sinks)
        if c > 1:
            seen[n - 1] = False  # the last token's own: the others are checked
        hold[page[seen], :, place[seen]] = False
    keys[hold] = bad
    values[hold] = bad
    got, want, tol = attend(dev, kind, batch, q, keys, values, window, sinks)
    for s in range(3):
        rows = slice(int(batch.starts[s]), int(batch.starts[s + 1]) - (1 if batch.new[s] > 1 else 0))
        assert not np.isnan(got[rows]).any()
        assert (np.abs(got[rows] - want[rows]).max(-1) <= tol[rows]).all()
        if batch.new[s] > 1:
            assert np.isnan(got[rows.stop]).any()


@pytest.mark.parametrize("kind", ["F32", "BF16"])
def test_infinities_that_are_seen(dev, kind):
    say("seen", kind)
    batch = ref.Batch([(1, 300), (40, 100)], 16, seed=9)
    q, keys, values = inputs(10, batch, 4, 2, 64)
    page, place = batch.slots(1)
    values[page[70], 0, place[70], 5] = np.inf
    values[page[80], 1, place[80], 6] = -np.inf
    values[page[90], 1, place[90], 6] = np.inf
    page, place = batch.slots(0)
    values[page[10], 0, place[10], 3] = np.nan
    keys[page[200], 1, place[200]] = 3e38  # a score past f32, or its opposite
    got, want, _ = attend(dev, kind, batch, q, keys, values)
    page, place = batch.slots(0)
    plain = np.isfinite(want)
    with np.errstate(invalid="ignore", over="ignore"):
        # the 64-bit form has scores that f32 has not
        score = (q[0].astype(np.float32) * keys[page[200], 1, place[200]]).sum(-1)
    plain[0, 2:] = False
    assert np.array_equal(np.isfinite(got)[1:], plain[1:])
    assert np.array_equal(got[1:][np.isinf(want[1:])], want[1:][np.isinf(want[1:])])
    assert np.isnan(got[0, :2, 3]).all() and np.isfinite(got[0, :2, 4:]).all()
    assert score.shape == (4,)


def test_index_errors(dev):
    batch = ref.Batch([(1, 100), (2, 40), (1, 50)], 16, seed=10)
    q, keys, values = inputs(11, batch, 4, 2, 64)

    def run(table=None, starts=None, lengths=None, max_new=2, max_length=100):
        say("index error", max_new, max_length)
        cache, _, _ = cache_of(dev, "F16", batch, 2, keys, values)
        b = dev.paged_batch(dev.from_array(batch.table if table is None else table), batch.table_width, 3,
                            dev.from_array(batch.starts if starts is None else np.array(starts, np.int32)),
                            dev.from_array(np.array(batch.lengths if lengths is None else lengths, np.int32)), max_new,
                            max_length)
        dst = dev.from_array(np.full(q.shape, 7.25, np.float32))
        dev.attention_paged(dev.from_array(q), batch.tokens, 4, cache, b, 0.125, dst=dst)
        got = dev.to_array(dst, np.float32, q.size).reshape(q.shape)
        with pytest.raises(th.ExecutionError):
            dev.sync()
        dev.sync()
        return got

    want, _ = ref.attention(q, *(ref.to_kind(a, "F16")[1] for a in (keys, values)), batch, 0.125)
    for bad in (-1, batch.pages, 2 ** 31 - 1):
        table = batch.table.copy()
        table[1, 1] = bad
        got = run(table=table)
        assert np.allclose(got[0], want[0], atol=1e-4) and np.allclose(got[3], want[3], atol=1e-4)
    for arrays in (dict(lengths=[100, 1, 50]), dict(lengths=[100, -5, 50]), dict(lengths=[100, 113, 50]),
                   dict(max_new=1), dict(starts=[0, 1, 5, 4])):
        got = run(**arrays)
        assert np.allclose(got[0], want[0], atol=1e-4)
        if "starts" not in arrays:
            assert (got[1:3] == 7.25).all() and np.allclose(got[3], want[3], atol=1e-4)
    got = run(max_length=60)
    assert (got[0] == 7.25).all() and np.allclose(got[1:], want[1:], atol=1e-4)


def test_strided_rows(dev):
    batch = ref.Batch([(1, 60), (90, 90), (2, 30)], 16, seed=12)
    q, keys, values = inputs(13, batch, 4, 2, 64)
    cache, k, v = cache_of(dev, "F16", batch, 2, keys, values)
    row = 4 * 64
    wide_q = np.zeros((batch.tokens, row + 3), np.float32)  # rows no load can take aligned
    wide_q[:, :row] = q.reshape(batch.tokens, row)
    dst = dev.from_array(np.full((batch.tokens, row + 5), 7.25, np.float32))
    say("strided")
    dev.attention_paged(dev.from_array(wide_q), batch.tokens, 4, cache, batch.on(dev), 0.125, dst=dst, ldq=row + 3,
                        ld_dst=row + 5)
    got = dev.to_array(dst, np.float32, batch.tokens * (row + 5)).reshape(batch.tokens, row + 5)
    dev.sync()
    assert (got[:, row:] == 7.25).all()
    want, tol = ref.attention(q, k, v, batch, 0.125)
    agree(got[:, :row].reshape(q.shape), want, tol, batch)


# ------------------------------------------------------------------ the writes

def tables(rows, width):
    angle = np.arange(rows)[:, None] / 10000.0 ** (np.arange(0, width, 2) / width)
    angle = np.concatenate([angle, angle], -1)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


@pytest.mark.parametrize("kind", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("heads,kv,width", HEADS)
@pytest.mark.parametrize("page_size", [16, 5])
def test_writes(dev, kind, heads, kv, width, page_size):
    say("write", kind, heads, kv, width, page_size)
    batch = ref.Batch([(1, 1), (1, 60), (0, 7), (30, 45), (8, 8)], page_size, seed=14, lead=1, trail=2)
    rng = np.random.default_rng(15)
    units = heads + 2 * kv
    ldx = units * width + 3
    x = rng.normal(0, 2, (batch.tokens, ldx)).astype(np.float32)
    cos, sin = tables(60, width)
    fill = np.full((batch.pages, kv, page_size, width), 3.0, np.float32)
    cache, k, v = cache_of(dev, kind, batch, kv, fill, fill)
    q = dev.from_array(np.full((batch.tokens, heads, width), 7.25, np.float32))
    dev.rope_write_paged(dev.from_array(x), ldx, batch.tokens, heads, dev.from_array(cos), dev.from_array(sin), 60, cache,
                         batch.on(dev), q_dst=q)
    got_q = dev.to_array(q, np.float32, batch.tokens * heads * width).reshape(batch.tokens, heads, width)
    raw = [dev.to_array(b, np.uint8, b.bytesize) for b in (cache.keys, cache.values)]
    got_k, got_v = (ref.from_bits(a, kind).reshape(fill.shape) for a in raw)
    dev.sync()
    want_q = np.full(got_q.shape, 7.25, np.float32)
    want_k, want_v = k.copy(), v.copy()
    for s, (c, n) in enumerate(zip(batch.new, batch.lengths)):
        rows = slice(int(batch.starts[s]), int(batch.starts[s]) + c)
        part = x[rows, :units * width].reshape(c, units, width)
        turned = ref.rope(part, cos[n - c:n], sin[n - c:n])
        page, place = batch.slots(s)
        want_q[rows] = turned[:, :heads]
        want_k[page[n - c:], :, place[n - c:]] = ref.to_kind(turned[:, heads:heads + kv], kind)[1]
        want_v[page[n - c:], :, place[n - c:]] = ref.to_kind(part[:, heads + kv:], kind)[1]
    for got, want in ((got_q, want_q), (got_k, want_k), (got_v, want_v)):
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


def test_write_index_errors(dev):
    batch = ref.Batch([(2, 20), (1, 30)], 16, seed=16)
    x = np.random.default_rng(17).normal(0, 1, (3, 4 * 64)).astype(np.float32)
    cos, sin = tables(30, 64)
    fill = np.full((batch.pages, 1, 16, 64), 3.0, np.float32)

    def run(table=None, rows=30, lengths=None):
        say("write index error", rows, lengths)
        cache, k, _ = cache_of(dev, "F32", batch, 1, fill, fill)
        b = dev.paged_batch(dev.from_array(batch.table if table is None else table), batch.table_width, 2,
                            dev.from_array(batch.starts),
                            dev.from_array(np.array(batch.lengths if lengths is None else lengths, np.int32)), 2, 30)
        dev.rope_write_paged(dev.from_array(x), 4 * 64, 3, 2, dev.from_array(cos), dev.from_array(sin), rows, cache, b)
        got = dev.to_array(cache.keys, np.float32, fill.size).reshape(fill.shape)
        with pytest.raises(th.ExecutionError):
            dev.sync()
        dev.sync()
        return got

    table = batch.table.copy()
    table[0, 1] = batch.pages
    page, place = batch.slots(1)
    for got in (run(table=table), run(lengths=[1, 30]), run(lengths=[33, 30])):
        assert (got[page[29], 0, place[29]] != 3.0).any()  # the other sequence's is written
        assert int((got != 3.0).any(-1).sum()) == 1
    assert int((run(rows=20) != 3.0).any(-1).sum()) == 2  # position 29 has no rotation


# ------------------------------------------------------- together, as a server

def test_a_server_of_three_sequences(dev):
    """Prompts in one batch, then steps: each position's queries, keys and values through the paged operators equal
    the same through the cache of fixed rows (its attention has other roundings: the tolerance of the attention), and
    the sampler picks from what a head gives."""
    heads, kv, width, vocab, ps = 6, 2, 64, 500, 16
    units = heads + 2 * kv
    rng = np.random.default_rng(18)
    prompt, steps = [37, 5, 18], 4
    cos, sin = tables(64, width)
    bcos, bsin = dev.from_array(cos), dev.from_array(sin)
    whole = ref.Batch([(0, n + steps) for n in prompt], ps, seed=19)
    cache = dev.paged_cache("F32", whole.pages, ps, kv, width)
    embed = rng.normal(0, 1, (vocab, units * width)).astype(np.float32)
    head = rng.normal(0, 0.3, (heads * width, vocab)).astype(np.float32)
    ids = [list(rng.integers(0, vocab, n)) for n in prompt]
    table = dev.from_array(whole.table)
    keys, values = dev.alloc(3 * kv * 64 * width * 4), dev.alloc(3 * kv * 64 * width * 4)
    new = list(prompt)
    for step in range(steps):
        say("server step", step)
        lengths = [len(i) for i in ids]
        starts = np.cumsum([0] + new).astype(np.int32)
        tokens = int(starts[-1])
        x = dev.from_array(np.concatenate([embed[i[n - c:]] for i, c, n in zip(ids, new, lengths)]))
        batch = dev.paged_batch(table, whole.table_width, 3, dev.from_array(starts),
                                dev.from_array(np.array(lengths, np.int32)), max(new), max(lengths))
        q = dev.rope_write_paged(x, units * width, tokens, heads, bcos, bsin, 64, cache, batch)
        out = dev.attention_paged(q, tokens, heads, cache, batch, 0.125)
        got = dev.to_array(out, np.float32, tokens * heads * width).reshape(tokens, heads, width)
        # the same over rows of 64 positions
        at = [(s, n - c + i) for s, (c, n) in enumerate(zip(new, lengths)) for i in range(c)]
        q2 = dev.alloc(tokens * heads * width * 4)
        dev.rope_write(x, units * width, tokens, heads, kv, width, bcos, bsin, 64,
                       dev.from_array(np.array([s * 64 + p for s, p in at], np.int32)), 3, 64, q2, keys, values)
        entries = np.array([(s, p, lengths[s]) for s, p in at], np.int32)
        out2 = dev.attention(q2, tokens, heads, keys, values, 3, kv, 64, width, dev.from_array(entries), 0.125)
        want = dev.to_array(out2, np.float32, tokens * heads * width).reshape(tokens, heads, width)
        assert np.array_equal(dev.to_array(q, np.uint32, tokens * heads * width),
                              dev.to_array(q2, np.uint32, tokens * heads * width))
        whole.new, whole.lengths, whole.starts = new, lengths, starts
        kk, vv = (dev.to_array(b, np.float32, b.bytesize // 4).reshape(whole.pages, kv, ps, width)
                  for b in (cache.keys, cache.values))
        qq = dev.to_array(q, np.float32, tokens * heads * width).reshape(tokens, heads, width)
        exact, tol = ref.attention(qq, kk, vv, whole, 0.125)
        assert (np.abs(got - exact).max(-1) <= tol).all() and (np.abs(got - want).max(-1) <= 2 * tol).all()
        logits = (got[starts[1:] - 1].reshape(3, -1) @ head).astype(np.float32)
        u, t = np.array([0.1, 0.5, 0.9], np.float32), np.array([0.7, 0.0, 1.2], np.float32)
        top = np.array([5, 0, 0], np.int32)
        p = np.array([1.0, 1.0, 0.8], np.float32)
        chosen = dev.to_array(dev.sample(dev.from_array(logits), 3, vocab, dev.from_array(u), dev.from_array(t),
                                         dev.from_array(top), dev.from_array(p)), np.int32, 3)
        dev.sync()
        for s in range(3):
            assert chosen[s] == ref.sample(logits[s], u[s], t[s], top[s], p[s])
            ids[s].append(int(chosen[s]))
        new = [1, 1, 1]


# ------------------------------------------------ what a caller may do besides

@pytest.mark.parametrize("kind", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("count,length", [(1, 1), (40, 40), (3, 1000), (200, 1000), (64, 64), (65, 129)])
@pytest.mark.parametrize("width", [64, 128])
def test_one_sequence_of_any_count(dev, kind, count, length, width):
    # one sequence alone, with max_new well above what it has
    say("one sequence", kind, count, length, width)
    batch = ref.Batch([(count, length)], 16, seed=30, lead=3, trail=5)
    q, keys, values = inputs(31, batch, 4, 2, width)
    cache, k, v = cache_of(dev, kind, batch, 2, keys, values)
    b = batch.on(dev)
    b.max_new, b.max_length = 300, 5000
    dst = dev.from_array(np.full(q.shape, 7.25, np.float32))
    dev.attention_paged(dev.from_array(q), batch.tokens, 4, cache, b, 0.125, dst=dst)
    got = dev.to_array(dst, np.float32, q.size).reshape(q.shape)
    dev.sync()
    want, tol = ref.attention(q, k, v, batch, 0.125)
    agree(got, want, tol, batch)


@pytest.mark.parametrize("kind", ["F32", "F16", "BF16"])
def test_many_heads_of_one_kv_head(dev, kind):
    # a single token's query rows fill more than a tile of few rows
    say("heads", kind)
    batch = ref.Batch([(1, 70), (1, 300), (3, 65)], 32, seed=32)
    for heads in (17, 33, 71):
        q, keys, values = inputs(33, batch, heads, 1, 64)
        agree(*attend(dev, kind, batch, q, keys, values), batch)


def test_pages_of_hidden_positions_may_be_gone(dev):
    # a server frees what has left the window: those entries are no pages, and are not looked at
    window, sinks, ps = 40, 5, 16
    for sequences in ([(1, 700), (1, 200), (20, 333), (90, 400)], [(100, 600)]):
        say("gone", sequences)
        batch = ref.Batch(sequences, ps, seed=34)
        q, keys, values = inputs(35, batch, 4, 2, 64)
        full = batch.table.copy()
        for s, (c, n) in enumerate(sequences):
            seen = np.zeros(n, bool)
            for i in range(c):
                seen |= ref.visible(n - c + i, np.arange(n), window, sinks)
            for page in range(-(-n // ps)):
                if not seen[page * ps:(page + 1) * ps].any():
                    batch.table[s, page] = -1
        assert (batch.table != full).any()
        cache, k, v = cache_of(dev, "F16", batch, 2, keys, values)
        dst = dev.from_array(np.full(q.shape, 7.25, np.float32))
        dev.attention_paged(dev.from_array(q), batch.tokens, 4, cache, batch.on(dev), 0.125, window=window, sinks=sinks,
                            dst=dst)
        got = dev.to_array(dst, np.float32, q.size).reshape(q.shape)
        dev.sync()  # no index error
        batch.table = full
        want, tol = ref.attention(q, k, v, batch, 0.125, window, sinks)
        agree(got, want, tol, batch)


def test_new_tokens_where_none_were_announced(dev):
    batch = ref.Batch([(1, 20), (1, 30)], 16, seed=36)
    q, keys, values = inputs(37, batch, 4, 2, 64)
    cache, _, _ = cache_of(dev, "F16", batch, 2, keys, values)
    for alone in (False, True):
        say("unannounced", alone)
        b = batch.on(dev)
        b.max_new = 0
        if alone:
            b.sequences, b.max_new, b.max_length = 1, 40, 19
        dst = dev.from_array(np.full(q.shape, 7.25, np.float32))
        dev.attention_paged(dev.from_array(q), batch.tokens, 4, cache, b, 0.125, dst=dst)
        got = dev.to_array(dst, np.float32, q.size)
        with pytest.raises(th.ExecutionError):
            dev.sync()
        assert (got == 7.25).all()


@pytest.mark.parametrize("kind,width", [("F32", 256), ("F16", 128)])
def test_a_cache_past_four_gigabytes(dev, kind, width):
    # pages at both ends of keys and values of more than 2^32 bytes each, and of more than 2^31 elements
    ps, size = 64, 4 if kind == "F32" else 2
    pages = (1 << 32) // (ps * width * size) + 400
    say("past 4 GB", kind, width, pages)
    batch = ref.Batch([(1, 150), (40, 200)], ps, seed=38, spare=0)
    q, keys, values = inputs(39, batch, 2, 1, width)
    small, k, v = cache_of(dev, kind, batch, 1, keys, values)
    big = dev.paged_cache(kind, pages, ps, 1, width)
    page = ps * width * size
    where = np.array([0, pages - 1, pages - 2, 1, pages - 5, pages - 3, pages - 4], np.int32)[:batch.pages]
    for i, at in enumerate(where):
        for name in ("keys", "values"):
            dev.copy(getattr(big, name), getattr(small, name), page, dst_offset=int(at) * page, src_offset=i * page)
    want, tol = ref.attention(q, k, v, batch, 0.125)
    held = batch.table.copy()
    batch.table = np.where(held >= 0, where[np.maximum(held, 0)], held).astype(np.int32)
    dst = dev.from_array(np.full(q.shape, 7.25, np.float32))
    dev.attention_paged(dev.from_array(q), batch.tokens, 2, big, batch.on(dev), 0.125, dst=dst)
    got = dev.to_array(dst, np.float32, q.size).reshape(q.shape)
    agree(got, want, tol, batch)
    # and a write there
    x = np.random.default_rng(40).normal(0, 1, (batch.tokens, 4 * width)).astype(np.float32)
    cos, sin = tables(200, width)
    dev.rope_write_paged(dev.from_array(x), 4 * width, batch.tokens, 2, dev.from_array(cos), dev.from_array(sin), 200, big,
                         batch.on(dev))
    last, place = batch.slots(1)
    out = dev.alloc(page)
    dev.copy(out, big.values, page, src_offset=int(last[199]) * page)
    row = ref.from_bits(dev.to_array(out, np.uint8, page), kind).reshape(ps, width)[place[199]]
    dev.sync()
    assert np.array_equal(row, ref.to_kind(x[-1, 3 * width:], kind)[1])
    limit = dev.counters()["pool_limit"]
    dev.set_pool_limit(0)  # so that the memory is given back
    for b in (big.keys, big.values):
        b.release()
    dev.sync()
    dev.set_pool_limit(limit)


def test_the_same_bits_on_every_call(dev):
    batch = ref.Batch([(1, 3000), (1, 700), (200, 900)], 16, seed=41)
    q, keys, values = inputs(42, batch, 8, 2, 64)
    first = None
    for _ in range(4):
        say("again")
        got, _, _ = attend(dev, "F16", batch, q, keys, values, window=500, sinks=4)
        first = got if first is None else first
        assert np.array_equal(got.view(np.uint32), first.view(np.uint32))


def test_two_threads(dev):
    # both need the library's scratch, of different sizes
    import threading
    jobs = []
    for seed, sequences, heads in ((50, [(1, 5000), (1, 200)], 4), (51, [(120, 2000), (1, 900)], 8)):
        batch = ref.Batch(sequences, 16, seed=seed)
        q, keys, values = inputs(seed, batch, heads, 2, 64)
        cache, k, v = cache_of(dev, "F16", batch, 2, keys, values)
        jobs.append((batch, heads, cache, dev.from_array(q), q.shape, ref.attention(q, k, v, batch, 0.125)))
    wrong = []

    def work(job):
        batch, heads, cache, q, shape, (want, tol) = job
        dev.bind()
        b = batch.on(dev)
        for _ in range(10):
            out = dev.attention_paged(q, batch.tokens, heads, cache, b, 0.125)
            got = dev.to_array(out, np.float32, int(np.prod(shape))).reshape(shape)
            if not (np.abs(got - want).max(-1) <= tol).all():
                wrong.append(heads)

    say("threads")
    threads = [threading.Thread(target=work, args=(job,)) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not wrong and not any(t.is_alive() for t in threads)
    dev.sync()


def test_no_memory_and_no_kernels(dev):
    # a growth of the scratch that fails is an error, and the next call has its scratch: this
    # call's parts, 4096 x 8 rows of 256 in two, are more than any other test's here
    tokens, heads, width, ps = 4096, 8, 256, 512
    batch = ref.Batch([(tokens, tokens)], ps, seed=52)
    zeros = dev.from_array(np.zeros((batch.pages, heads, ps, width), np.float16))
    cache = dev.paged_cache("F16", batch.pages, ps, heads, width, keys=zeros, values=zeros)
    q = np.random.default_rng(53).normal(0, 1, (tokens, heads, width)).astype(np.float32)
    b, qb, dst = batch.on(dev), dev.from_array(q), dev.from_array(np.ones_like(q))
    say("no memory")
    dev.lib.tmh_debug_disable_kernels(1)
    try:
        with pytest.raises(th.NoKernels):
            dev.attention_paged(qb, tokens, heads, cache, b, 0.125, dst=dst)
    finally:
        dev.lib.tmh_debug_disable_kernels(0)
    dev.lib.tmh_debug_fail_allocations(1)
    try:
        with pytest.raises(th.DeviceError, match="OUT_OF_MEMORY"):
            dev.attention_paged(qb, tokens, heads, cache, b, 0.125, dst=dst)
    finally:
        dev.lib.tmh_debug_fail_allocations(0)
    assert (dev.to_array(dst, np.float32, q.size) == 1.0).all()
    dev.attention_paged(qb, tokens, heads, cache, b, 0.125, dst=dst)
    got = dev.to_array(dst, np.float32, q.size)
    dev.sync()
    assert (got == 0.0).all()


@pytest.mark.parametrize("kind", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("heads,kv,width", [(4, 2, 32), (2, 1, 64), (4, 1, 128), (2, 2, 256)])
def test_steps_and_chunks_split_in_one_call(dev, kind, heads, kv, width):
    # row tiles and few rows of one launch, both in parts that one launch joins
    say("split", kind, heads, kv, width)
    batch = ref.Batch([(1, 5000), (64, 4100), (0, 12), (3, 2700), (130, 3333)], 32, seed=31, lead=1, trail=2)
    q, keys, values = inputs(32, batch, heads, kv, width)
    agree(*attend(dev, kind, batch, q, keys, values), batch)
    agree(*attend(dev, kind, batch, q, keys, values, window=1500, sinks=70), batch)


def test_more_sequences_than_a_wave_has_lanes(dev):
    say("sequences")
    rng = np.random.default_rng(33)
    sizes = [(int(rng.choice([0, 1, 1, 2, 40])), 0) for _ in range(200)]
    sizes = [(n, n + int(rng.integers(0, 60))) for n, _ in sizes]
    batch = ref.Batch(sizes, 8, seed=34, lead=3, trail=1)
    q, keys, values = inputs(35, batch, 4, 2, 64)
    agree(*attend(dev, "F16", batch, q, keys, values), batch)


def test_pages_that_two_sequences_share(dev):
    # a common prefix: the first four pages of one table are the other's
    say("shared")
    batch = ref.Batch([(5, 100), (40, 90)], 16, seed=36)
    batch.table[1, :4] = batch.table[0, :4]
    q, keys, values = inputs(37, batch, 4, 2, 64)
    agree(*attend(dev, "BF16", batch, q, keys, values), batch)


@pytest.mark.parametrize("max_new,max_length", [(500, 4000), (500, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("sizes", [[(1, 20), (2, 133)], [(9, 9)], [(60, 300), (1, 1000)]])
def test_loose_bounds(dev, max_new, max_length, sizes):
    # announced: more new tokens and longer sequences than there are
    say("loose", max_new, max_length, sizes)
    batch = ref.Batch(sizes, 16, seed=38, lead=1)
    q, keys, values = inputs(39, batch, 4, 2, 64)
    cache, k, v = cache_of(dev, "F16", batch, 2, keys, values)
    b = batch.on(dev)
    b.max_new, b.max_length = max_new, max_length
    dst = dev.from_array(np.full(q.shape, 7.25, np.float32))
    dev.attention_paged(dev.from_array(q), batch.tokens, 4, cache, b, 0.125, dst=dst)
    got = dev.to_array(dst, np.float32, q.size).reshape(q.shape)
    dev.sync()
    agree(got, *ref.attention(q, k, v, batch, 0.125), batch)
