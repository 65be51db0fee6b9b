"""Refused calls of the serving operators, without a GPU: arguments are checked
before the device is asked for, so a good call says that there is no GPU (or,
on one with a GPU, is not made)."""
import numpy as np
import pytest

import paged_reference as ref
import tensomite_hip as th

P = 1 << 20  # an address that no call here reaches


def write(x=P, ldx=7 * 64, tokens=4, heads=3, kv=2, width=64, cos=P, sin=P, rows=50, kind=1, pages=9, page_size=16,
          table=P, table_width=4, sequences=2, starts=P, lengths=P, q=P, keys=P, values=P):
    return th.library().tmh_rope_write_paged(x, ldx, tokens, heads, kv, width, cos, sin, rows, kind, pages, page_size,
                                             table, table_width, sequences, starts, lengths, q, keys, values)


def attend(q=P, ldq=6 * 64, tokens=4, heads=6, kind=1, keys=P, values=P, pages=9, page_size=16, kv=2, width=64,
           table=P, table_width=4, sequences=2, starts=P, lengths=P, max_new=4, max_length=60, window=0, sinks=0,
           scale=0.125, dst=P, ld_dst=6 * 64):
    return th.library().tmh_attention_paged(q, ldq, tokens, heads, kind, keys, values, pages, page_size, kv, width,
                                            table, table_width, sequences, starts, lengths, max_new, max_length,
                                            window, sinks, scale, dst, ld_dst)


def sample(x=P, ldx=100, rows=3, n=100, t=P, k=P, p=P, m=P, u=P, ids=P):
    return th.library().tmh_sample(x, ldx, rows, n, t, k, p, m, u, ids)


SHAPE, VALUE, DTYPE = th.ERROR_SHAPE, th.ERROR_INVALID_VALUE, th.ERROR_DTYPE
CACHE = [(dict(kind=2), DTYPE), (dict(kind=8), DTYPE), (dict(width=0), SHAPE), (dict(width=12), SHAPE),
         (dict(width=264), SHAPE), (dict(kv=0), SHAPE), (dict(pages=0), SHAPE), (dict(page_size=0), SHAPE),
         (dict(table_width=0), SHAPE), (dict(pages=1 << 20, page_size=1 << 10), SHAPE), (dict(tokens=1 << 24), SHAPE),
         (dict(tokens=1 << 31), SHAPE),
         (dict(sequences=1 << 16, table_width=1 << 15), SHAPE), (dict(keys=0), VALUE), (dict(values=0), VALUE),
         (dict(keys=P + 8), VALUE), (dict(values=P + 2), VALUE), (dict(table=0), VALUE), (dict(starts=0), VALUE),
         (dict(lengths=0), VALUE)]


@pytest.mark.parametrize("change,code", CACHE + [
    (dict(ldx=7 * 64 - 1), SHAPE), (dict(heads=0), SHAPE), (dict(rows=0), SHAPE), (dict(x=0), VALUE),
    (dict(cos=0), VALUE), (dict(sin=0), VALUE), (dict(q=0), VALUE), (dict(tokens=0), 0), (dict(sequences=0), 0)])
def test_write(change, code):
    assert write(**change) == code


@pytest.mark.parametrize("change,code", CACHE + [
    (dict(heads=0), SHAPE), (dict(heads=5), SHAPE), (dict(ldq=6 * 64 - 1), SHAPE), (dict(ld_dst=63), SHAPE),
    (dict(max_new=1 << 31), SHAPE), (dict(max_length=1 << 31), SHAPE), (dict(window=1 << 31), SHAPE),
    (dict(sinks=1 << 31), SHAPE), (dict(q=0), VALUE), (dict(dst=0), VALUE), (dict(tokens=0), 0),
    (dict(sequences=0), 0), (dict(tokens=1 << 30), SHAPE)])
def test_attention(change, code):
    assert attend(**change) == code


@pytest.mark.parametrize("change,code", [
    (dict(n=0), SHAPE), (dict(ldx=99), SHAPE), (dict(n=(1 << 24) + 1, ldx=1 << 25), SHAPE), (dict(rows=1 << 31), SHAPE),
    (dict(x=0), VALUE), (dict(u=0), VALUE), (dict(ids=0), VALUE), (dict(rows=0), 0)])
def test_sample(change, code):
    assert sample(**change) == code


def test_good_calls_ask_for_a_gpu():
    import torch
    if torch.cuda.is_available():
        pytest.skip("the calls would run")
    for call in (write, attend, sample):
        assert call() == th.ERROR_NO_DEVICE


class Device(th.HIPDevice):
    """The binding's checks without a GPU."""

    def __init__(self):
        self.lib = th.library()

    def buffer(self, bytesize):
        b = th.Buffer(self, P, bytesize)
        b._released = True
        return b


def test_binding_refuses_small_buffers():
    dev = Device()
    b = dev.buffer
    with pytest.raises(th.DTypeError):
        dev.paged_cache("Q8_0", 4, 16, 2, 64)
    size = 4 * 16 * 2 * 64 * 2
    cache = dev.paged_cache("F16", 4, 16, 2, 64, keys=b(size), values=b(size))
    assert cache.code == 1
    for keys, values in ((size - 1, size), (size, size - 1)):
        with pytest.raises(th.ShapeError):
            dev.paged_cache("F16", 4, 16, 2, 64, keys=b(keys), values=b(values))
    for table, starts, lengths in ((31, 12, 8), (32, 11, 8), (32, 12, 7)):
        with pytest.raises(th.ShapeError):
            dev.paged_batch(b(table), 4, 2, b(starts), b(lengths), 1, 64)
    batch = dev.paged_batch(b(32), 4, 2, b(12), b(8), 1, 64)
    row = 8 * 64 * 4
    good = dict(x=b(2 * row), ldx=8 * 64, tokens=2, heads=4, cos=b(50 * 256), sin=b(50 * 256), table_rows=50, cache=cache,
                batch=batch, q_dst=b(2 * 4 * 64 * 4))
    for name, less in (("x", 2 * row - 1), ("cos", 50 * 256 - 1), ("sin", 50 * 256 - 1), ("q_dst", 2 * 4 * 64 * 4 - 1)):
        with pytest.raises(th.ShapeError):
            dev.rope_write_paged(**dict(good, **{name: b(less)}))
    size = 2 * 4 * 64 * 4
    for q, dst in ((size - 1, size), (size, size - 1)):
        with pytest.raises(th.ShapeError):
            dev.attention_paged(b(q), 2, 4, cache, batch, 0.125, dst=b(dst))
    for x, u, ids in ((3999, 40, 40), (4000, 39, 40), (4000, 40, 39)):
        with pytest.raises(th.ShapeError):
            dev.sample(b(x), 10, 100, b(u), ids=b(ids))


def test_reference_by_hand():
    # the plain forms that the GPU's results are held to
    assert ref.sample([1.0, 3.0, 2.0], 0.0) == 1
    assert ref.sample([1.0, 3.0, 2.0], 0.999) == 0
    assert ref.sample([1.0, 3.0, 2.0], 0.999, k=2) == 2
    assert ref.sample([1.0, 3.0, 2.0], 0.999, p=0.6) == 1  # 0.665 alone reaches it
    assert ref.sample([1.0, 3.0, 2.0], 0.999, p=0.7) == 2
    assert ref.sample([1.0, 3.0, 2.0], 0.999, m=0.3) == 2  # e^-1 = 0.37 stays, e^-2 = 0.14 does not
    assert ref.sample([1.0, 1.0, 1.0, 1.0], 0.5) == 2
    assert ref.sample([5.0, 5.0], 0.9, t=0.0) == 0
    batch = ref.Batch([(2, 3)], 2, spare=0)
    q = np.zeros((2, 1, 8), np.float32)
    values = np.zeros((2, 1, 2, 8), np.float32)
    page, place = batch.slots(0)
    for p in range(3):
        values[page[p], 0, place[p]] = 3.0 ** p
    out, _ = ref.attention(q, values, values, batch, 1.0)
    assert np.allclose(out[0], 2.0) and np.allclose(out[1], 13.0 / 3.0)
    out, _ = ref.attention(q, values, values, batch, 1.0, window=1, sinks=1)
    assert np.allclose(out[0], 2.0) and np.allclose(out[1], 5.0)
