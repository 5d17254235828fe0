"""Dropout against the generator restated on the host: the same bits, at any stride."""
import ctypes as C

import numpy as np
import pytest
import torch

import lm_ref as R


def test_generator_known_answers():
    """The published vectors of Philox-4x32-10 (all counters and keys zero; all ones)."""
    zero = R.philox(*[np.zeros(1, np.uint64)] * 4, 0, 0)
    assert [int(x[0]) for x in zero] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = R.philox(*[np.full(1, 0xFFFFFFFF, np.uint64)] * 4, 0xFFFFFFFF, 0xFFFFFFFF)
    assert [int(x[0]) for x in ones] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def expected(x, res, p, seed, offset, dtype):
    """One multiply and one add in binary32, one rounding to the type; raw bytes."""
    keep, up = R.keep_mask(x.size, p, seed, offset)
    x32 = x.astype(np.float32)
    y = np.where(keep.reshape(x.shape), x32 * up, np.float32(0))
    if res is not None:
        y = res.astype(np.float32) + y
    return R.bytes_of(y.astype(np.float32), dtype)


def run(gm, dev, x, res, p, seed, offset, dtype, ld_x, ld_r, ld_y, shift=0, offset_device=0):
    rows, cols = x.shape
    eb = R.eb(dtype)

    def put(a, ld):
        raw = np.zeros(rows * ld * eb + 64, np.uint8)
        b = R.bytes_of(R.strided(a, ld, dtype), dtype)
        raw[shift * eb:shift * eb + b.size] = b
        return dev.to_device(raw)
    dx = put(x, ld_x)
    dr = put(res, ld_r) if res is not None else 0
    dy = put(np.zeros_like(x), ld_y)
    at = shift * eb
    gm.check(gm.lib.gm_dropout_async(dev.h, dtype, rows, cols, dx + at, ld_x, dr + at if dr else 0, ld_r, dy + at, ld_y,
                                     gm.dropout(p, seed, offset, offset_device)), "dropout")
    raw = dev.to_host(dy, rows * ld_y * eb + 64, np.uint8)
    for b in (dx, dr, dy):
        if b:
            dev.free(b)
    body = raw[at:at + rows * ld_y * eb].reshape(rows, ld_y * eb)
    gap = R.values_of(body[:, cols * eb:].copy().reshape(-1), dtype)
    assert np.all(gap == -7.0), "columns behind the row were written"
    assert not raw[:at].any() and not raw[at + rows * ld_y * eb:].any(), "bytes around the matrix were written"
    return body[:, :cols * eb].reshape(-1)


SHAPES = [(1, 1), (1, 7), (3, 8), (5, 13), (16, 1000), (2, 4097), (301, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [0, 2, 4])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_bits(gm, dev, dtype, shape, p, residual):
    rng = np.random.default_rng(shape[0] * 1000 + shape[1])
    x = R.rounded(rng.standard_normal(shape), dtype)
    res = R.rounded(rng.standard_normal(shape), dtype) if residual else None
    c = shape[1]
    want = expected(x, res, p, 0x123456789ABCDEF0, 7, dtype)
    for ld_x, ld_r, ld_y, shift in [(c, c, c, 0), (c + 8, c + 16, c + 8, 0), (c + 3, c, c + 5, 0), (c, c, c, 1)]:
        got = run(gm, dev, x, res, p, 0x123456789ABCDEF0, 7, dtype, ld_x, ld_r, ld_y, shift)
        assert np.array_equal(got, want), (ld_x, ld_r, ld_y, shift)


@pytest.mark.gpu
def test_dropped_nan_and_infinity_are_dropped(gm, dev):
    x = np.full((4, 64), np.nan)
    x[1] = np.inf
    got = R.values_of(run(gm, dev, x, None, 0.5, 3, 0, 0, 64, 64, 64), 0).reshape(4, 64)
    keep, _ = R.keep_mask(256, 0.5, 3, 0)
    keep = keep.reshape(4, 64)
    assert np.all(got[~keep] == 0) and np.all(~np.isfinite(got[keep]))


@pytest.mark.gpu
def test_backward_is_the_same_mask_and_offsets_differ(gm, dev):
    x = np.ones((32, 128))
    a = run(gm, dev, x, None, 0.3, 11, 4, 2, 128, 128, 128)
    b = run(gm, dev, x, None, 0.3, 11, 4, 2, 136, 128, 128)
    c = run(gm, dev, x, None, 0.3, 11, 5, 2, 128, 128, 128)
    assert np.array_equal(a, b) and not np.array_equal(a, c)
    kept = np.count_nonzero(R.values_of(a, 2))
    assert abs(kept - 0.7 * 4096) < 6 * np.sqrt(4096 * 0.21)       # six standard deviations


@pytest.mark.gpu
def test_device_offset_is_added_with_carry(gm, dev):
    x = np.ones((4, 40))
    word = dev.to_device(np.array([0xFFFFFFFF], np.uint64))
    got = run(gm, dev, x, None, 0.5, 5, 3, 0, 40, 40, 40, offset_device=word)
    assert np.array_equal(got, expected(x, None, 0.5, 5, 0xFFFFFFFF + 3, 0))
    dev.free(word)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [0, 4])
def test_in_place(gm, dev, dtype):
    rng = np.random.default_rng(1)
    x, res = R.rounded(rng.standard_normal((9, 48)), dtype), R.rounded(rng.standard_normal((9, 48)), dtype)
    want = expected(x, res, 0.25, 1, 2, dtype)
    for target in ("x", "res"):
        dx, dr = dev.to_device(R.bytes_of(x, dtype)), dev.to_device(R.bytes_of(res, dtype))
        y = dx if target == "x" else dr
        gm.check(gm.lib.gm_dropout_async(dev.h, dtype, 9, 48, dx, 48, dr, 48, y, 48, gm.dropout(0.25, 1, 2)), "dropout")
        assert np.array_equal(dev.to_host(y, want.size, np.uint8), want)
        dev.free(dx)
        dev.free(dr)


@pytest.mark.gpu
def test_replayed_graph_goes_on_with_the_device_offset(gm, dev):
    """A captured call reads the offset when it runs: two replays with another word, two masks."""
    n = 512
    x = torch.ones(n, device="cuda")
    y = torch.empty(n, device="cuda")
    word = torch.zeros(1, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.ExternalStream(gm.lib.gm_device_stream(dev.h))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        gm.check(gm.lib.gm_dropout_async(dev.h, 0, 1, n, x.data_ptr(), n, 0, n, y.data_ptr(), n, gm.dropout(0.5, 9, 100, word.data_ptr())))
    for k in (0, 1, 77):
        word.fill_(k)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(y.cpu().numpy() != 0, R.keep_mask(n, 0.5, 9, 100 + k)[0])


@pytest.mark.gpu
def test_refusals(gm, dev):
    L, ok = gm.lib, gm.dropout(0.1, 1)
    b = dev.alloc(4 * 64)
    before = L.gm_device_launch_count(dev.h)

    def call(rc, dtype=0, rows=4, cols=16, x=b, ld_x=16, r=0, ld_r=16, y=b, ld_y=16, d=ok, h=None):
        assert L.gm_dropout_async(dev.h if h is None else h, dtype, rows, cols, x, ld_x, r, ld_r, y, ld_y, d) == rc, gm.last_error()
        assert gm.last_error()
    call(-1, h=0)
    call(-10, dtype=1)
    call(-10, dtype=3)
    call(-10, d=None)
    call(-10, d=gm.dropout(-0.1, 1))
    call(-10, d=gm.dropout(1.5, 1))
    call(-10, d=gm.dropout(float("nan"), 1))
    call(-10, d=gm.dropout(0.1, 1, 0, 4))
    call(-9, rows=0)
    call(-9, cols=0)
    call(-9, rows=-1)
    call(-9, rows=1 << 31)
    call(-9, rows=(1 << 31) - 1, ld_x=1 << 40)
    call(-10, ld_x=15)
    call(-10, ld_y=15)
    call(-10, r=b, ld_r=3)
    call(-4, x=0)
    call(-4, y=0)
    call(-9, rows=5)
    call(-9, ld_y=17)
    call(-10, x=b + 2)
    call(-10, rows=2, ld_x=24)                  # in place with another stride
    assert L.gm_device_launch_count(dev.h) == before
    dev.free(b)


@pytest.mark.gpu
def test_refuses_a_device_offset_shorter_than_a_word(gm, dev):
    b, word = dev.alloc(4 * 64), dev.alloc(4)
    before = gm.lib.gm_device_launch_count(dev.h)
    assert gm.lib.gm_dropout_async(dev.h, 0, 4, 16, b, 16, 0, 16, b, 16, gm.dropout(0.1, 1, 0, word)) == -9
    assert gm.last_error() and gm.lib.gm_device_launch_count(dev.h) == before
    dev.free(b)
    dev.free(word)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [0, 2, 4])
@pytest.mark.parametrize("rows,cols,ld", [(200, 13, 15), (64, 4091, 4091), (64, 4091, 4093), (40, 1000, 1001)])
def test_in_place_at_odd_addresses(gm, dev, dtype, rows, cols, ld):
    """Groups of eight share 16-byte words with their neighbours there, which other threads write meanwhile."""
    rng = np.random.default_rng(cols)
    x, res = R.rounded(rng.standard_normal((rows, cols)), dtype), R.rounded(rng.standard_normal((rows, cols)), dtype)
    want = expected(x, res, 0.25, 1, 2, dtype)
    eb = R.eb(dtype)
    for target in ("x", "res"):
        dx, dr = (dev.to_device(np.concatenate([np.zeros(eb, np.uint8), R.bytes_of(R.strided(a, ld, dtype), dtype), np.zeros(64, np.uint8)])) for a in (x, res))
        y = dx if target == "x" else dr
        gm.check(gm.lib.gm_dropout_async(dev.h, dtype, rows, cols, dx + eb, ld, dr + eb, ld, y + eb, ld, gm.dropout(0.25, 1, 2)), "dropout")
        got = dev.to_host(y, eb + rows * ld * eb + 64, np.uint8)
        assert not got[:eb].any() and not got[eb + rows * ld * eb:].any(), "bytes around the matrix were written"
        body = got[eb:eb + rows * ld * eb].reshape(rows, ld * eb)
        assert np.array_equal(body[:, :cols * eb].reshape(-1), want)
        assert np.all(R.values_of(body[:, cols * eb:].copy().reshape(-1), dtype) == -7.0), "columns behind the row were written"
        dev.free(dx)
        dev.free(dr)
