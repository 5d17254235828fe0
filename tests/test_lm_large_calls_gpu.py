"""Forms of the language-model operators that only larger calls take, against 64 bits on the device: more sorted words per
chunk and a third and fourth merge in the lookup's gradient, several tokens per thread in the lookup, dX and dW in launches
of their own in the vocabulary loss, and losses to a bound near their real error."""
import numpy as np
import pytest
import torch

import lm_ref as R
from test_linear_xent_gpu import Call, check_backward, check_forward, make, reference

F32, F16, BF16 = 0, 2, 4
SCALE = 1.75
U = 2.0 ** -24


def P(t):
    return t.data_ptr()


def strided(rows, cols, extra, shift, dtype, fill):
    """A matrix inside a larger buffer, `shift` elements off a 16-byte boundary, and the whole buffer."""
    ld = cols + extra
    flat = torch.full((shift + rows * ld + 64,), fill, dtype=R.TORCH[dtype], device="cuda")
    return torch.as_strided(flat, (rows, cols), (ld, 1), shift), flat


def power_law(n, vocab, g):
    rank = torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * np.log(vocab + 1)).long() - 1
    return torch.randperm(vocab, generator=g, device="cuda")[rank.clamp(0, vocab - 1)].int()


def runs_of(lengths, n, g):
    """Tokens, in any order, of which the first values occur `lengths` times each, again and again."""
    again = torch.tensor(lengths * (n // sum(lengths) + 1), device="cuda")
    t = torch.repeat_interleave(torch.arange(len(again), device="cuda"), again)[:n]
    return t[torch.randperm(n, generator=g, device="cuda")].int()


# tokens x columns / 8: below 1,212,416 eight words per chunk, below 2,424,832 sixteen, then 32
LARGE = [(13001, 800, 16), (70001, 72, 8), (40000, 261, 16), (20000, 1024, 32), (69000, 288, 32), (66000, 296, 32), (1300000, 8, 16), (40001, 501, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,dim,words", LARGE)
@pytest.mark.parametrize("dtype,gdtype,kind,extra,shift,p,accumulate", [
    (F16, F16, "runs", 0, 0, 0.0, 0), (BF16, F32, "power", 0, 0, 0.3, 1), (F32, F32, "runs", 0, 0, 0.0, 1), (F32, F32, "power", 3, 1, 0.3, 0),
    (BF16, BF16, "runs", 5, 1, 0.3, 1), (F16, F32, "same", 8, 0, 0.0, 0)])
def test_table_gradient(gm, dev, n, dim, words, dtype, gdtype, kind, extra, shift, p, accumulate):
    """A row of L tokens takes at most L + L / 8 + 2 additions in binary32 and two multiplications, each off by U of what it
    holds, at most the sum of magnitudes; then one rounding to the type."""
    walks = n * ((dim + 7) // 8)
    assert words == (32 if walks >= 32 * 148 * 512 else 16 if walks >= 16 * 148 * 512 else 8)
    g = torch.Generator(device="cuda").manual_seed(n + dim)
    if kind == "runs":
        lengths = [31, 1, 32, 33, 15, 16, 17, 64, 7, 8, 9, 95, 1, 1, 200, 3]
        tok = runs_of(lengths, n, g)
        vocab = int(tok.max()) + 3
    elif kind == "power":
        vocab = 5003
        tok = power_law(n, vocab, g)
        tok[::97] = -5
        tok[5::101] = vocab
    else:
        vocab = 40
        tok = torch.full((n,), 7, dtype=torch.int32, device="cuda")
        tok[n // 2] = 3
    padding = int(tok[1]) if accumulate else -1
    dout, keep_dout = strided(n, dim, extra, shift, dtype, 3.0)
    dout.copy_(torch.randn(n, dim, generator=g, device="cuda"))
    grad, whole = strided(vocab, dim, extra, shift, gdtype, -7.0)
    grad.copy_(torch.randn(vocab, dim, generator=g, device="cuda"))
    base, around = grad.double(), whole.clone()
    e = gm.Embedding(dtype=dtype, tokens=n, dim=dim, vocab=vocab, ld_table=dim + extra, ld_out=dim + extra, padding_token=padding, scale=SCALE)
    size = gm.lib.gm_embedding_workspace_bytes(e)
    room = torch.full((size + 256,), 0xA5, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()

    def call():
        gm.check(gm.lib.gm_embedding_backward_async(dev.h, e, P(tok), P(dout), gm.dropout(p, 5, 9) if p else None, P(grad), gdtype, accumulate, P(room), size))
        dev.sync()
    call()
    x = dout.double()
    if p:
        keep, up = R.keep_mask(n * dim, p, 5, 9)
        x = x * torch.from_numpy(keep).cuda().view(n, dim) * float(up)
    x *= SCALE
    t = tok.long()
    ok = (t >= 0) & (t < vocab) & (t != padding)
    want, mags = torch.zeros(vocab, dim, dtype=torch.float64, device="cuda"), torch.zeros(vocab, dim, dtype=torch.float64, device="cuda")
    count = torch.zeros(vocab, dtype=torch.float64, device="cuda")
    want.index_add_(0, t[ok], x[ok])
    mags.index_add_(0, t[ok], x[ok].abs())
    count.index_add_(0, t[ok], torch.ones_like(t[ok], dtype=torch.float64))
    del x
    if accumulate:
        want, mags = want + base, mags + base.abs()
        empty = count == 0
        assert torch.equal(grad.double()[empty], base[empty]), "a row without tokens was changed"
        want[empty] = base[empty]
    steps = (count + count / 8 + 5)[:, None]
    bound = steps * U * 1.01 * mags + R.HALF_STEP[gdtype] * (want.abs() + steps * U * mags) + R.TINY[gdtype]
    got = grad.clone()
    assert torch.all((got.double() - want).abs() <= bound), float(((got.double() - want).abs() / bound).max())
    grad.copy_(base)
    assert torch.equal(whole, around), "something around the gradient was written"
    assert bool((room[size:] == 0xA5).all()), "the workspace was overrun"
    torch.cuda.synchronize()
    call()
    assert torch.equal(grad, got), "the same call gave other bits"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,dim,extra,shift", [(2501, 1024, 0, 0), (2501, 1024, 8, 0), (2502, 1003, 0, 0), (2503, 1024, 1, 1), (38003, 40, 0, 0), (38001, 13, 3, 1),
                                               (1203, 2048, 16, 0), (600, 4099, 1, 0)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_lookup_of_many_tokens(gm, dev, dtype, n, dim, extra, shift, p):
    """Bits: one multiplication in binary32 by scale times dropout's factor, one rounding."""
    vocab = 3001
    g = torch.Generator(device="cuda").manual_seed(n)
    tok = torch.randint(-5, vocab + 5, (n,), generator=g, device="cuda", dtype=torch.int32)
    table, keep_table = strided(vocab, dim, extra, shift, dtype, 9.0)
    table.copy_(torch.randn(vocab, dim, generator=g, device="cuda"))
    out, whole = strided(n, dim, extra, shift, dtype, -7.0)
    around = whole.clone()
    e = gm.Embedding(dtype=dtype, tokens=n, dim=dim, vocab=vocab, ld_table=dim + extra, ld_out=dim + extra, padding_token=2, scale=SCALE)
    torch.cuda.synchronize()
    gm.check(gm.lib.gm_embedding_forward_async(dev.h, e, P(table), P(tok), P(out), gm.dropout(p, 77, 1 << 40) if p else None))
    dev.sync()
    ok = (tok >= 0) & (tok < vocab)
    rows = table[torch.where(ok, tok, torch.zeros_like(tok)).long()].float()
    keep, up = R.keep_mask(n * dim, p, 77, 1 << 40)
    stays = torch.from_numpy(keep).cuda().view(n, dim) & ok[:, None]
    want = torch.where(stays, rows * float(np.float32(SCALE) * np.float32(up)), torch.zeros_like(rows)).to(R.TORCH[dtype])
    assert torch.equal(out, want)
    out.fill_(-7.0)
    assert torch.equal(whole, around), "something around the output was written"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,dim,vocab,extra", [(2600, 4096, 16700, 0), (2570, 4092, 17000, 3)])
def test_gradients_in_launches_of_their_own(gm, dev, dtype, n, dim, vocab, extra):
    """More than 16 rounds of tiles, dX in more than two: both gradients asked for, one launch each."""
    tiles = lambda k: (k + 255) // 256
    assert (tiles(n) + tiles(vocab)) * tiles(dim) > 16 * 74 and tiles(n) * tiles(dim) > 2 * 74
    x, w, t = make(dtype, n, dim, vocab, 3, 0.02)
    call = Call(gm, dev, dtype, x, w, t, 1, extra)
    ref, err, count = reference(x, w, t, 1.0)
    check_forward(call.forward(), ref, err, count, 1)
    got = call.backward(grad_scale=float(count))
    check_backward(got, ref, err, call)
    # in the 2-norm, where the roundings to the type of S and of the result, each at most half a step, add up at random
    half = R.HALF_STEP[dtype]
    for a, b in zip(got, (ref["dx"], ref["dw"])):
        assert np.linalg.norm(a - b) <= 1.5 * half * np.linalg.norm(b)
    call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,dim,vocab", [(100, 1024, 3000), (300, 1024, 3000), (1100, 512, 2000), (50, 2048, 1500), (200, 2056, 1500)])
def test_losses_to_their_real_error(gm, dev, dtype, n, dim, vocab):
    """A logit of the tensor cores: 16 products and the sum so far, 17 numbers of which each is cut below 2^-25 of the largest,
    2^-21 of (|sum so far| + the step's magnitudes) a step.  The target's: 128 chains of D / 128 binary32 additions, joined
    by 9 more, (D / 128 + 9) U of the sum of magnitudes.  The log-sum-exp weighs the logits' errors with the probabilities;
    its own: 8 exponentials (2^-22), arguments rounded (1.5 U times the distance to the maximum, 7 times), 64 additions."""
    x, w, t = make(dtype, n, dim, vocab, n + dim, 0.1)
    call = Call(gm, dev, dtype, x, w, t)
    losses, lse, total = call.forward()
    call.close()
    steps = (dim + 15) // 16
    X, W = torch.zeros(n, steps * 16, dtype=torch.float64, device="cuda"), torch.zeros(vocab, steps * 16, dtype=torch.float64, device="cuda")
    X[:, :dim], W[:, :dim] = torch.from_numpy(x).cuda(), torch.from_numpy(w).cuda()
    l, size = torch.zeros(n, vocab, dtype=torch.float64, device="cuda"), torch.zeros(n, vocab, dtype=torch.float64, device="cuda")
    for k in range(steps):
        a, b = X[:, 16 * k:16 * k + 16], W[:, 16 * k:16 * k + 16]
        l += a @ b.T
        size += l.abs() + a.abs() @ b.abs().T
    ok = torch.from_numpy((t >= 0)).cuda()
    at = torch.from_numpy(np.maximum(t, 0).astype(np.int64)).cuda()[:, None]
    p = torch.softmax(l, 1)
    want_lse = torch.logsumexp(l, 1)
    z = l.gather(1, at)[:, 0]
    want = want_lse - z
    spread = (p * (l.max(1, keepdim=True).values - l)).sum(1)
    own = (X.abs() * W.abs()[at[:, 0]]).sum(1)
    e_z = (dim / 128 + 9) * U * own
    e_lse = 2.0 ** -21 * (p * size).sum(1) + p.gather(1, at)[:, 0] * e_z + 2.0 ** -22 * 8 + 10.5 * U * spread + 64 * U + 4 * U * (want_lse.abs() + 1)
    bound = e_lse + e_z + 4 * U * (want.abs() + 1)
    got, got_lse = torch.from_numpy(losses).cuda().double(), torch.from_numpy(lse).cuda().double()
    assert torch.all((got - want).abs()[ok] <= bound[ok]), float(((got - want).abs() / bound)[ok].max())
    assert torch.all((got_lse - want_lse).abs()[ok] <= e_lse[ok])
    assert bool((bound[ok] < 2.0 ** -11).all())                       # the bound is worth something
    mean = float(want[ok].mean())
    assert abs(float(total[0]) - mean) <= float(bound[ok].mean()) + 9 * U * mean
    # errors of either sign average out over the rows, but for the cut's, which goes one way: half its bound
    assert float(((got - want)[ok] ** 2).mean().sqrt()) <= float((bound[ok] ** 2).mean().sqrt()) / 2
