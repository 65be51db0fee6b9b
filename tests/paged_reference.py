"""The serving operators in 64 bits with numpy, and batches to try them on."""
import math

import numpy as np

EPS = 2.0 ** -24  # half a step of f32, relative


def to_kind(a, kind):
    """(the array as the cache holds it, the values it stands for)."""
    a = np.ascontiguousarray(a, np.float32)
    if kind == "F32":
        return a, a
    if kind == "F16":
        with np.errstate(over="ignore"):
            h = a.astype(np.float16)
        return h, h.astype(np.float32)
    bits = a.view(np.uint32).astype(np.uint64)
    nan = np.isnan(a)
    r = ((bits + 0x7fff + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    r = np.where(nan, np.uint16(0x7fc0), r)
    return r, (r.astype(np.uint32) << 16).view(np.float32)


def from_bits(raw, kind):
    """Values of a downloaded cache."""
    if kind == "BF16":
        return (raw.view(np.uint16).astype(np.uint32) << 16).view(np.float32)
    return raw.view(np.float16).astype(np.float32) if kind == "F16" else raw.view(np.float32)


class Batch:
    """Sequences of (new tokens, positions), on pages in no order; `lead` rows belong to none of them."""

    def __init__(self, sequences, page_size, seed=0, lead=0, trail=0, spare=2):
        self.new = [c for c, _ in sequences]
        self.lengths = [n for _, n in sequences]
        self.page_size = page_size
        per = [-(-n // page_size) for n in self.lengths]
        self.pages = max(1, sum(per) + spare)
        order = np.random.default_rng(seed).permutation(self.pages)
        self.table_width = max(1, max(per, default=1))
        self.table = np.full((len(per), self.table_width), -7, np.int32)  # unread entries are no pages
        at = 0
        for s, count in enumerate(per):
            self.table[s, :count] = order[at:at + count]
            at += count
        self.starts = (np.cumsum([0] + self.new) + lead).astype(np.int32)
        self.tokens = int(self.starts[-1]) + trail

    def slots(self, s):
        """(page, place) of the positions of sequence s."""
        at = np.arange(self.lengths[s])
        return self.table[s][at // self.page_size], at % self.page_size

    def on(self, dev):
        return dev.paged_batch(dev.from_array(self.table), self.table_width, len(self.new),
                               dev.from_array(self.starts), dev.from_array(np.array(self.lengths, np.int32)),
                               max(self.new, default=0), max(self.lengths, default=0))


def visible(pos, j, window, sinks):
    return (j <= pos) & ((window == 0) | (pos - j < window) | (j < sinks))


def attention(q, keys, values, batch, scale, window=0, sinks=0):
    """(outputs [tokens, heads, width] in f64 with NaN in rows of no sequence, tolerance per row and head).

    The tolerance: each of the width roundings of a score's sum is off by at
    most EPS of the sum of its terms' magnitudes, A; they fall either way, so
    3.5 sqrt(width) of them (six standard deviations of an even spread) plus 8
    for the scale, the splits of q and the exponential's argument bound a
    score's error in units of EPS A. A score's error moves its weight by that
    much of it, an output by at most twice that of the largest value. The
    weights' exponential (1 step), their splits (4) and the sums over n
    positions in runs of at least 32 (3.5 sqrt(n / 32) + 32) come on top."""
    tokens, heads, width = q.shape
    group = heads // keys.shape[1]
    out = np.full(q.shape, np.nan)
    tol = np.zeros((tokens, heads))
    for s, (c, n) in enumerate(zip(batch.new, batch.lengths)):
        page, place = batch.slots(s)
        first = int(batch.starts[s])
        for h in range(heads):
            k = keys[page, h // group, place].astype(np.float64)
            v = values[page, h // group, place].astype(np.float64)
            for i in range(c):
                see = visible(n - c + i, np.arange(n), window, sinks)
                with np.errstate(all="ignore"):
                    x = q[first + i, h].astype(np.float64)
                    score = k[see] @ x * scale
                    e = np.exp(score - score.max())
                    out[first + i, h] = (e / e.sum()) @ v[see]
                    a = (np.abs(k[see]) @ np.abs(x)).max() * abs(scale)
                    count = int(see.sum())
                    tol[first + i, h] = EPS * np.abs(v[see]).max() * (
                        2 * a * (3.5 * math.sqrt(width) + 8) + 3.5 * math.sqrt(count / 32) + 64)
    return out, tol


def rope(x, cos, sin):
    """x [tokens, units, width] rotated, in f32 as the device's other RoPE rounds it."""
    half = x.shape[-1] // 2
    turned = np.concatenate([x[..., half:] * np.float32(-1), x[..., :half]], -1)
    return x * cos[:, None] + turned * sin[:, None]


def sample(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """The next token of one row, by sorting it."""
    x = np.asarray(x, np.float32)
    ok = np.flatnonzero(x == x)
    if not t > 0 or not (x[ok] > -np.inf).any():
        if x[0] != x[0] or ok.size == 0:
            return 0
        return int(ok[np.argmax(x[ok])])
    order = ok[np.lexsort((ok, -x[ok].astype(np.float64)))]
    if 0 < k < order.size:
        order = order[:k]
    z = x[order].astype(np.float64)
    with np.errstate(invalid="ignore"):
        w = np.exp(np.where(z == z[0], 0.0, (z - z[0]) / np.float64(np.float32(t))))
    total = w.sum()
    if not np.float32(p) >= 1.0:
        before = np.cumsum(w) - w
        stay = before < np.float64(np.float32(p)) * total
        stay[0] = True
        order, w = order[stay], w[stay]
    stay = w >= np.float64(np.float32(m))
    stay[0] = True
    order, w = order[stay], w[stay]
    target = np.float64(np.float32(u)) * w.sum()
    above = np.flatnonzero(np.cumsum(w) > target)
    return int(order[above[0] if above.size else np.flatnonzero(w)[-1]])
