"""Sampling on the GPU against the definition by sorting, in 64 bits: equal ids."""
import numpy as np
import pytest

import paged_reference as ref
import tensomite_hip as th

pytestmark = pytest.mark.gpu


def say(*args):
    print(*args, flush=True)


@pytest.fixture(scope="module")
def dev():
    return th.HIPDevice(0)


def settings(rng, rows):
    """Rows of settings, every step on and off."""
    t = rng.choice([0.0, 0.3, 0.8, 1.0, 1.7, 10.0], rows).astype(np.float32)
    k = rng.choice([0, 1, 2, 40, 1000, 10 ** 9, -3], rows).astype(np.int32)
    p = rng.choice([1.0, 0.0, 0.1, 0.5, 0.9, 0.999, 2.0], rows).astype(np.float32)
    m = rng.choice([0.0, 0.01, 0.2, 1.0, 3.0], rows).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    u[::7] = 0.0
    u[3::7] = np.float32(1.0) - np.float32(2.0 ** -24)
    return u, t, k, p, m


def run(dev, x, u, t=None, k=None, p=None, m=None, ldx=None, rows=None, n=None):
    rows = x.shape[0] if rows is None else rows
    n = x.shape[1] if n is None else n
    up = lambda a: None if a is None else dev.from_array(a)  # noqa: E731
    ids = dev.sample(dev.from_array(x), rows, n, up(u), temperature=up(t), top_k=up(k), top_p=up(p), min_p=up(m),
                     ldx=ldx)
    got = dev.to_array(ids, np.int32, rows)
    dev.sync()
    return got


@pytest.mark.parametrize("n,rows", [(1, 20), (2, 40), (63, 60), (1000, 80), (4097, 60), (49152, 24), (50257, 16),
                                    (131072, 12), (300001, 5)])
@pytest.mark.parametrize("spread", [0.3, 3.0])
def test_ids(dev, n, rows, spread):
    say("sample", n, rows, spread)
    rng = np.random.default_rng(n + int(10 * spread))
    x = rng.normal(0, spread, (rows, n)).astype(np.float32)
    u, t, k, p, m = settings(rng, rows)
    got = run(dev, x, u, t, k, p, m)
    want = [ref.sample(x[r], u[r], t[r], k[r], p[r], m[r]) for r in range(rows)]
    assert list(got) == want


@pytest.mark.parametrize("which", ["none", "t", "k", "p", "m"])
def test_arrays_left_out(dev, which):
    say("left out", which)
    rng = np.random.default_rng(5)
    x = rng.normal(0, 2, (30, 3001)).astype(np.float32)
    u, t, k, p, m = settings(rng, 30)
    given = {"t": t, "k": k, "p": p, "m": m}
    given = {name: a for name, a in given.items() if name == which}
    got = run(dev, x, u, **given)
    full = {"t": np.ones(30), "k": np.zeros(30, int), "p": np.ones(30), "m": np.zeros(30), **given}
    assert list(got) == [ref.sample(x[r], u[r], *(full[name][r] for name in "tkpm")) for r in range(30)]


@pytest.mark.parametrize("n", [300, 1500, 9000, 40000])
def test_ties(dev, n):
    # few values many times over, and one value only: equal candidates by rising index
    say("ties", n)
    rng = np.random.default_rng(n)
    rows = 36
    x = rng.integers(-3, 4, (rows, n)).astype(np.float32)
    x[::3] = np.where(rng.random((12, n)) < 0.5, np.float32(0.0), np.float32(-0.0))
    x[1::3] = np.float32(2.5) + rng.integers(0, 3, (12, n)).astype(np.float32) * np.float32(2.0 ** -22)
    u, t, k, p, m = settings(rng, rows)
    k = np.where(k > 2, rng.integers(1, n + 1, rows), k).astype(np.int32)
    got = run(dev, x, u, t, k, p, m)
    assert list(got) == [ref.sample(x[r], u[r], t[r], k[r], p[r], m[r]) for r in range(rows)]


def test_many_close_values(dev):
    # one bin of the histogram with more values than are put in order at once, all different
    say("close")
    rng = np.random.default_rng(8)
    rows, n = 12, 30000
    x = (np.float32(1.0) + rng.permutation(n).astype(np.float32) * np.float32(2.0 ** -23))[None].repeat(rows, 0)
    x[:, 0] = -30.0
    x[:, 1] = 1.0 + 2.0 ** -6
    u = rng.random(rows).astype(np.float32)
    t = np.full(rows, 1.0, np.float32)
    k = np.array([0, 5, 3000, 20000] * 3, np.int32)
    p = np.array([1.0, 0.5, 0.9] * 4, np.float32)
    got = run(dev, x, u, t, k, p)
    assert list(got) == [ref.sample(x[r], u[r], t[r], k[r], p[r]) for r in range(rows)]


def test_masked_and_odd_logits(dev):
    say("masked")
    rng = np.random.default_rng(9)
    n = 2000
    x = rng.normal(0, 2, (12, n)).astype(np.float32)
    x[0, 5:] = -np.inf
    x[1] = -np.inf
    x[1, 1234] = -80.0
    x[2] = -np.inf                          # nothing left: the greedy choice
    x[3] = np.nan
    x[4, ::2] = np.nan
    x[5, 17] = np.inf
    x[6, [100, 900]] = np.inf
    x[7] = np.finfo(np.float32).min         # masks of the type's lowest value
    x[7, 50:60] = 1.0
    x[8] = np.finfo(np.float32).min
    x[9] = np.finfo(np.float32).max
    x[10, 0] = np.nan
    x[11] *= 1e30
    for trial in range(6):
        u, t, k, p, m = settings(rng, 12)
        got = run(dev, x, u, t, k, p, m)
        assert list(got) == [ref.sample(x[r], u[r], t[r], k[r], p[r], m[r]) for r in range(12)]


def test_random_numbers_out_of_range(dev):
    say("range")
    x = np.array([[0.0, 3.0, 1.0, 2.0]] * 4, np.float32)
    got = run(dev, x, np.array([1.0, 7.0, -1.0, np.nan], np.float32))
    assert list(got) == [0, 0, 1, 0]  # the last that stays, the last, the first, the last
    got = run(dev, x, np.array([1.0, 0.99, 0.99, 0.99], np.float32), k=np.array([2, 2, 3, 1], np.int32))
    assert list(got) == [3, 3, 2, 1]


def test_strided_rows_and_the_same_ids_again(dev):
    say("strided")
    rng = np.random.default_rng(11)
    x = rng.normal(0, 2, (9, 5003)).astype(np.float32)
    u, t, k, p, m = settings(rng, 9)
    got = run(dev, x, u, t, k, p, m, ldx=5003, rows=9, n=4999)
    assert list(got) == [ref.sample(x[r, :4999], u[r], t[r], k[r], p[r], m[r]) for r in range(9)]
    for _ in range(3):
        assert list(run(dev, x, u, t, k, p, m, ldx=5003, rows=9, n=4999)) == list(got)


def test_frequencies(dev):
    # 4096 even steps of u over one row: each token as often as its weight says, to one step
    say("frequencies")
    x = np.tile(np.log(np.array([0.5, 0.25, 0.15, 0.1], np.float32)), (4096, 1))
    u = ((np.arange(4096) + 0.5) / 4096).astype(np.float32)
    counts = np.bincount(run(dev, x, u), minlength=4)
    assert np.abs(counts - 4096 * np.array([0.5, 0.25, 0.15, 0.1])).max() <= 1.0


def test_no_temperature_is_argmax(dev):
    say("greedy")
    rng = np.random.default_rng(12)
    x = rng.integers(-4, 5, (40, 7001)).astype(np.float32)
    x[3, 0] = np.nan
    x[4] = np.nan
    x[5, 1:] = np.nan
    x[6] = -np.inf
    x[7, 100] = np.inf
    buf = dev.from_array(x)
    want = dev.to_array(dev.argmax(buf, 40, 7001), np.int32, 40)
    for t in (0.0, -1.0, np.nan):
        got = run(dev, x, np.full(40, 0.7, np.float32), np.full(40, t, np.float32), k=np.full(40, 9, np.int32))
        assert list(got) == list(want)


def test_rows_past_four_gigabytes(dev):
    rows, n, ldx = 3, 5000, 700000000
    say("past 4 GB")
    rng = np.random.default_rng(13)
    x = rng.normal(0, 2, (rows, n)).astype(np.float32)
    big, small = dev.alloc(4 * ((rows - 1) * ldx + n)), dev.from_array(x)
    for r in range(rows):
        dev.copy(big, small, 4 * n, dst_offset=4 * r * ldx, src_offset=4 * r * n)
    u = np.array([0.2, 0.5, 0.9], np.float32)
    got = dev.to_array(dev.sample(big, rows, n, dev.from_array(u), ldx=ldx), np.int32, rows)
    dev.sync()
    assert list(got) == [ref.sample(x[r], u[r]) for r in range(rows)]
    limit = dev.counters()["pool_limit"]
    dev.set_pool_limit(0)  # so that the memory is given back
    big.release()
    dev.sync()
    dev.set_pool_limit(limit)


def test_lists_of_every_length(dev):
    # top-k at the sizes where the candidates change hands: a wave's, the list's, the histogram's finer ones
    say("lists")
    rng = np.random.default_rng(14)
    n = 60000
    x = rng.normal(0, 3, n).astype(np.float32)
    k = np.array([1, 2, 63, 64, 65, 66, 255, 1023, 1024, 1025, 4000, 4095, 4096, 4097, 8000, 59999], np.int32)
    rows = k.size
    x = np.stack([rng.permutation(x) for _ in range(rows)])
    for u in (0.0, 0.37, 0.99, np.float32(1) - np.float32(2.0 ** -24)):
        for p in (1.0, 0.97):
            us, ps = np.full(rows, u, np.float32), np.full(rows, p, np.float32)
            for t in (0.5, 5.0):
                ts = np.full(rows, t, np.float32)
                got = run(dev, x, us, ts, k, ps)
                assert list(got) == [ref.sample(x[r], u, t, k[r], p) for r in range(rows)]


def odd_rows(rng, n):
    """Rows whose candidates, masks and ties fall in one part of them or across all."""
    x = rng.normal(0, 2, (14, n)).astype(np.float32)
    x[0] = -np.sort(-x[0])                      # the first ones next to each other
    x[1] = np.sort(x[1])
    x[2, : n - 100] = -np.inf
    x[3, 7:] = -np.inf
    x[4] = np.nan
    x[4, n // 2] = -3.0
    x[5, rng.permutation(n)[: n // 2]] = np.nan
    x[6, [5, n // 3, n - 1]] = np.inf
    x[7] = rng.integers(-2, 3, n)               # ties by the thousand
    x[8] = 1.25                                 # one value
    x[9] = np.float32(1.0) + rng.permutation(n).astype(np.float32) * np.float32(2.0 ** -23)
    x[9, 0], x[9, 1] = -30.0, 1.0 + 2.0 ** -4
    x[10] = np.finfo(np.float32).min
    x[10, n - 50:] = 1.0
    x[11] *= 1e30
    x[12] = 40.0 - 1e-3 * np.arange(n)          # most of them too far below to count
    x[13] = -np.inf
    return x


@pytest.mark.parametrize("n", [70003, 131072])
def test_rows_in_chunks(dev, n):
    # few long rows, which several workgroups share
    say("chunks", n)
    rng = np.random.default_rng(15)
    x = odd_rows(rng, n)
    rows = len(x)
    for trial in range(8):
        u, t, k, p, m = settings(rng, rows)
        if trial == 1:
            k[:], p[:], m[:] = 0, 1.0, 0.0
        if trial == 2:
            k[:], p[:], m[:] = 0, 0.95, 0.0
        if trial == 3:
            k[:], p[:], m[:] = 3000, 1.0, 0.0
        if trial == 4:
            k[:], p[:], m[:] = 40, 0.9, 0.05
        got = run(dev, x, u, t, k, p, m)
        assert list(got) == [ref.sample(x[r], u[r], t[r], k[r], p[r], m[r]) for r in range(rows)], trial


@pytest.mark.parametrize("n", [500, 70000])
def test_extreme_temperatures(dev, n):
    say("temperatures", n)
    rng = np.random.default_rng(16)
    t = np.array([1e-38, 1e-30, 1e-10, 1e10, 1e30, 3e38, np.inf, 1e-42], np.float32)
    rows = t.size
    x = rng.normal(0, 2, (rows, n)).astype(np.float32)
    x[:, 11] = x[:, 40] = x[:, n - 2] = 30.0    # three first ones
    x[4] *= 1e30
    for u in (0.0, 0.4, 0.99):
        for k, p in ((0, 1.0), (0, 0.9), (100, 1.0)):
            us, ks, ps = np.full(rows, u, np.float32), np.full(rows, k, np.int32), np.full(rows, p, np.float32)
            got = run(dev, x, us, t, ks, ps)
            assert list(got) == [ref.sample(x[r], us[r], t[r], k, ps[r]) for r in range(rows)], (u, k, p)
