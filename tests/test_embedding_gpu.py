"""Embedding lookup and its gradient against a plain restatement in 64 bits."""
import ctypes as C

import numpy as np
import pytest
import torch

import lm_ref as R

SCALE = 1.75                    # exact in binary32


def emb(gm, dtype, n, dim, vocab, ld_table=None, ld_out=None, padding=-1, scale=SCALE):
    return gm.Embedding(dtype=dtype, tokens=n, dim=dim, vocab=vocab, ld_table=ld_table or dim, ld_out=ld_out or dim,
                        padding_token=padding, scale=scale)


def put(dev, values, ld, dtype, shift=0):
    eb = R.eb(dtype)
    b = R.bytes_of(R.strided(values, ld, dtype), dtype)
    raw = np.zeros(b.size + 64, np.uint8)
    raw[shift * eb:shift * eb + b.size] = b
    return dev.to_device(raw)


def get(dev, p, rows, cols, ld, dtype, shift=0):
    """The matrix as float64; what lies around it must be as it was."""
    eb = R.eb(dtype)
    raw = dev.to_host(p, rows * ld * eb + 64, np.uint8)
    at = shift * eb
    assert not raw[:at].any() and not raw[at + rows * ld * eb:].any(), "bytes around the matrix were written"
    v = R.values_of(raw[at:at + rows * ld * eb].copy(), dtype).reshape(rows, ld)
    assert np.all(v[:, cols:] == -7.0), "columns behind the row were written"
    return v[:, :cols]


def tokens_of(kind, n, vocab, rng):
    if kind == "uniform":
        t = rng.integers(0, vocab, n)
    elif kind == "same":
        t = np.full(n, vocab - 1)
    elif kind == "power":
        t = np.minimum((np.exp(rng.random(n) * np.log(vocab + 1)) - 1).astype(np.int64), vocab - 1)
    elif kind == "runs":                       # runs whose ends fall around the sums' chunk borders
        t = np.sort(np.concatenate([np.full(k, j % vocab) for j, k in enumerate([63, 1, 64, 65, 128, 127, 1, 1, 200] * (n // 600 + 1))])[:n])
        t = rng.permutation(t)
    else:                                      # some tokens outside the table, on both sides
        t = rng.integers(-vocab, 2 * vocab, n)
    return t.astype(np.int32)


LAYOUTS = [(0, 0, 0), (8, 16, 0), (3, 5, 0), (0, 0, 1)]        # extra stride of table and out, elements of misalignment


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [0, 2, 4])
@pytest.mark.parametrize("n,dim,vocab", [(1, 1, 1), (3, 8, 5), (7, 13, 300), (130, 72, 1000), (33, 1000, 257), (2, 5000, 10)])
@pytest.mark.parametrize("p", [0.0, 0.4])
def test_forward(gm, dev, dtype, n, dim, vocab, p):
    rng = np.random.default_rng(n * dim)
    table = R.rounded(rng.standard_normal((vocab, dim)), dtype)
    tok = tokens_of("outside", n, vocab, rng)
    tok[0] = vocab - 1
    keep, up = R.keep_mask(n * dim, p, 77, 1 << 40)
    rows = np.where((tok >= 0) & (tok < vocab), tok, 0)
    want = table[rows].astype(np.float32) * (np.float32(SCALE) * up)
    want = np.where(keep.reshape(n, dim) & ((tok >= 0) & (tok < vocab))[:, None], want, np.float32(0))
    want = R.rounded(want.astype(np.float32), dtype)
    d_tok = dev.to_device(tok)
    for et, eo, shift in LAYOUTS:
        e = emb(gm, dtype, n, dim, vocab, dim + et, dim + eo)
        d_table, d_out = put(dev, table, dim + et, dtype, shift), put(dev, np.zeros((n, dim)), dim + eo, dtype, shift)
        at = shift * R.eb(dtype)
        gm.check(gm.lib.gm_embedding_forward_async(dev.h, e, d_table + at, d_tok, d_out + at, gm.dropout(p, 77, 1 << 40) if p else None))
        assert np.array_equal(get(dev, d_out, n, dim, dim + eo, dtype, shift), want), (et, eo, shift)
        dev.free(d_table)
        dev.free(d_out)
    dev.free(d_tok)


def backward(gm, dev, dtype, gdtype, tok, dout, vocab, p, padding, accumulate, base, extra=(0, 0, 0)):
    n, dim = dout.shape
    et, eo, shift = extra
    e = emb(gm, dtype, n, dim, vocab, dim + et, dim + eo, padding)
    d_tok, d_dout = dev.to_device(tok), put(dev, dout, dim + eo, dtype, shift)
    d_grad = put(dev, base, dim + et, gdtype, shift)
    size = gm.lib.gm_embedding_workspace_bytes(e)
    ws = dev.to_device(np.full(size + 256, 0xA5, np.uint8))
    gm.check(gm.lib.gm_embedding_backward_async(dev.h, e, d_tok, d_dout + shift * R.eb(dtype), gm.dropout(p, 5, 9) if p else None,
                                                d_grad + shift * R.eb(gdtype), gdtype, accumulate, ws, size))
    got = get(dev, d_grad, vocab, dim, dim + et, gdtype, shift)
    assert np.all(dev.to_host(ws, size + 256, np.uint8)[size:] == 0xA5), "the workspace was overrun"
    for b in (d_tok, d_dout, d_grad, ws):
        dev.free(b)
    return got


def check_backward(got, dtype, gdtype, tok, dout, vocab, p, padding, accumulate, base):
    """Within the error of a sum of L terms in binary32 and one rounding to the type: each of at most
    L + L/64 + 2 additions and the multiplications by scale and factor (2) is off by 2^-24 relative
    to what it holds, which is at most the sum of magnitudes."""
    n, dim = dout.shape
    keep, up = R.keep_mask(n * dim, p, 5, 9)
    factor = SCALE * float(up)
    x = np.where(keep.reshape(n, dim), dout, 0.0)
    ok = (tok >= 0) & (tok < vocab) & (tok != padding)
    want, size, count = np.zeros((vocab, dim)), np.zeros((vocab, dim)), np.zeros(vocab)
    np.add.at(want, tok[ok], x[ok] * factor)
    np.add.at(size, tok[ok], np.abs(x[ok]) * factor)
    np.add.at(count, tok[ok], 1)
    if accumulate:
        untouched = count == 0
        assert np.array_equal(got[untouched], base[untouched]), "a row without tokens was changed"
        want, size = want + base, size + np.abs(base)
        want[untouched] = base[untouched]
    steps = (count + count / 64 + 5)[:, None]
    bound = steps * 2.0 ** -24 * 1.01 * size + R.HALF_STEP[gdtype] * (np.abs(want) + steps * 2.0 ** -24 * size) + R.TINY[gdtype]
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) - bound))


CASES = [("uniform", 1, 1, 1), ("uniform", 5, 13, 3), ("outside", 64, 8, 40), ("outside", 65, 24, 40), ("same", 1000, 16, 7),
         ("runs", 1300, 40, 1000), ("power", 1025, 72, 5000), ("power", 5000, 136, 3000), ("same", 4096, 8, 300), ("outside", 33, 1000, 65)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gdtype", [(0, 0), (2, 2), (2, 0), (4, 4), (4, 0)])
@pytest.mark.parametrize("kind,n,dim,vocab", CASES)
@pytest.mark.parametrize("accumulate", [0, 1])
def test_backward(gm, dev, dtype, gdtype, kind, n, dim, vocab, accumulate):
    rng = np.random.default_rng(n * dim + vocab)
    tok = tokens_of(kind, n, vocab, rng)
    dout = R.rounded(rng.standard_normal((n, dim)), dtype)
    base = R.rounded(rng.standard_normal((vocab, dim)), gdtype)
    for p, padding, extra in [(0.0, -1, (0, 0, 0)), (0.3, int(tok[0]), (8, 16, 0)), (0.0, -1, (3, 1, 0)), (0.3, -1, (0, 0, 1))]:
        got = backward(gm, dev, dtype, gdtype, tok, dout, vocab, p, padding, accumulate, base, extra)
        check_backward(got, dtype, gdtype, tok, dout, vocab, p, padding, accumulate, base)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [32769, 40000])
def test_backward_of_many_tokens(gm, dev, n):
    """Beyond one merge of 32 sorted tiles; the same call twice gives the same bits."""
    rng = np.random.default_rng(n)
    tok = tokens_of("power", n, 4000, rng)
    dout = R.rounded(rng.standard_normal((n, 16)), 4)
    base = np.zeros((4000, 16))
    got = backward(gm, dev, 4, 0, tok, dout, 4000, 0.1, -1, 0, base)
    check_backward(got, 4, 0, tok, dout, 4000, 0.1, -1, 0, base)
    assert np.array_equal(got, backward(gm, dev, 4, 0, tok, dout, 4000, 0.1, -1, 0, base))


@pytest.mark.gpu
def test_nan_stays_in_its_row(gm, dev):
    """Rows of dout that padding or a token outside the table names may hold anything."""
    tok = np.array([3, 1, -1, 9, 3, 2], np.int32)
    dout = np.ones((6, 16))
    dout[2] = np.nan
    dout[3] = np.inf
    dout[1] = np.nan
    got = backward(gm, dev, 0, 0, tok, dout, 5, 0.0, 1, 0, np.zeros((5, 16)))
    assert np.all(np.isfinite(got)) and np.all(got[3] == 2 * SCALE) and np.all(got[1] == 0)


@pytest.mark.gpu
def test_gradient_against_differences(gm, dev):
    """The lookup is linear in the table: <dtable, D> equals the change of <dout, out> along D."""
    rng = np.random.default_rng(3)
    n, dim, vocab = 50, 24, 20
    tok = tokens_of("power", n, vocab, rng)
    table, direction, dout = rng.standard_normal((vocab, dim)), rng.standard_normal((vocab, dim)), R.rounded(rng.standard_normal((n, dim)), 0)
    e = emb(gm, 0, n, dim, vocab)
    drop = gm.dropout(0.2, 5, 9)
    outs = []
    for t in (table, table + direction):
        d_table, d_tok, d_out = dev.to_device(R.bytes_of(t, 0)), dev.to_device(tok), dev.alloc(n * dim * 4)
        gm.check(gm.lib.gm_embedding_forward_async(dev.h, e, d_table, d_tok, d_out, drop))
        outs.append(dev.to_host(d_out, n * dim).astype(np.float64).reshape(n, dim))
        for b in (d_table, d_tok, d_out):
            dev.free(b)
    grad = backward(gm, dev, 0, 0, tok, dout, vocab, 0.2, -1, 0, np.zeros((vocab, dim)))
    left, right = np.sum(grad * direction), np.sum(dout * (outs[1] - outs[0]))
    size = np.sum(np.abs(dout) * np.abs(outs[1] - outs[0])) + np.sum(np.abs(dout) * np.abs(outs[0]))
    assert abs(left - right) <= 64 * 2.0 ** -24 * size       # each output is three roundings off, each gradient at most n + 4


@pytest.mark.gpu
def test_refusals(gm, dev):
    L = gm.lib
    n, dim, vocab = 4, 16, 8
    e = emb(gm, 0, n, dim, vocab)
    size = L.gm_embedding_workspace_bytes(e)
    table, tok, out, ws = dev.alloc(vocab * dim * 4), dev.alloc(n * 4), dev.alloc(n * dim * 4), dev.alloc(size)
    before = L.gm_device_launch_count(dev.h)

    def fwd(rc, e=e, t=table, k=tok, o=out, d=None, h=None):
        assert L.gm_embedding_forward_async(dev.h if h is None else h, e, t, k, o, d) == rc, gm.last_error()

    def bwd(rc, e=e, k=tok, o=out, d=None, t=table, gd=0, w=ws, wb=size, h=None):
        assert L.gm_embedding_backward_async(dev.h if h is None else h, e, k, o, d, t, gd, 0, w, wb) == rc, gm.last_error()
    for call in (fwd, bwd):
        call(-1, h=0)
        call(-10, e=None)
        call(-10, e=emb(gm, 1, n, dim, vocab))
        call(-9, e=emb(gm, 0, 0, dim, vocab))
        call(-9, e=emb(gm, 0, n, 0, vocab, 16, 16))
        call(-9, e=emb(gm, 0, n, dim, -1))
        call(-9, e=emb(gm, 0, n, dim, (1 << 31) - 1))
        call(-10, e=emb(gm, 0, n, dim, vocab, 15))
        call(-10, e=emb(gm, 0, n, dim, vocab, 16, 15))
        call(-4, k=0)
        call(-4, t=0)
        call(-4, o=0)
        call(-9, e=emb(gm, 0, n + 1, dim, vocab))
        call(-9, e=emb(gm, 0, n, dim, vocab + 1))
        call(-10, d=gm.dropout(2.0, 1))
        call(-10, k=tok + 2)
    bwd(-10, gd=2)
    bwd(-9, wb=size - 1)
    bwd(-4, w=0)
    bwd(-10, w=ws + 128)
    assert L.gm_device_launch_count(dev.h) == before
    for b in (table, tok, out, ws):
        dev.free(b)


def test_workspace_size_needs_no_device(gm):
    assert gm.lib.gm_embedding_workspace_bytes(emb(gm, 0, 4, 16, 8)) > 0
    assert gm.lib.gm_embedding_workspace_bytes(emb(gm, 0, 4, 16, 8, 15)) == -1
    assert gm.lib.gm_embedding_workspace_bytes(emb(gm, 3, 4, 16, 8)) == -1
    assert gm.lib.gm_embedding_workspace_bytes(None) == -1
