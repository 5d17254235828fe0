"""The vocabulary loss where a model is sure of itself: statistics of large logits, small losses, and the
gradient of a target whose probability is nearly one, each against 64 bits."""
import numpy as np
import pytest
import torch

import lm_ref as R
from test_linear_xent_gpu import Call

F16, BF16 = 2, 4
U = 2.0 ** -24                       # half a unit in the last place of a binary32 number, relative


def exact_logits(n, vocab, mean, deviation, seed):
    """Hidden states and a table whose logits are sums of three products, all multiples of 2^-8 below 2^10: exact
    in binary32 in any order, so what is off comes from the row statistics.  Every second row's target stands
    14 to 29 above all other entries."""
    g = np.random.default_rng(seed)
    w = np.zeros((vocab, 8))
    w[:, 0] = np.round(g.standard_normal(vocab) * deviation * 128) / 128
    w[:, 1] = mean
    w[0, :3] = 0.0, mean, 1.0
    w = R.rounded(np.clip(w, -250, 250), F16)
    w[:, 0] = np.round(w[:, 0] * 128) / 128                      # fp16 holds multiples of 2^-7 up to 16, coarser ones beyond
    x = np.zeros((n, 8))
    x[:, 0] = g.choice([1.0, -1.0, 0.5, -0.5], n)
    x[:, 1] = 1.0
    t = g.integers(1, vocab, n).astype(np.int32)
    sure = np.arange(n) % 2 == 0
    t[sure] = 0
    rest = (x @ w.T)[:, 1:].max(1) - mean
    x[sure, 2] = np.ceil(rest[sure]) + g.integers(14, 30, sure.sum())
    return x, w, t, sure


@pytest.mark.gpu
@pytest.mark.parametrize("n,vocab", [(20, 20000), (100, 5003), (140, 50257), (1100, 131072), (1100, 700)])
@pytest.mark.parametrize("mean,deviation", [(0, 1), (0, 10), (200, 1), (-200, 10)])
def test_row_statistics_of_large_logits(gm, dev, n, vocab, mean, deviation):
    """Error of the sum of exponentials, relatively.  A term: the exponential 2^-22, its argument's rounding and
    that of log2(e), 1.5 U times the distance to the maximum.  A piece of 128: at most 32 additions and one factor for the
    reference (2^-22).  Joining: a lane has at most pieces / 32 of them, and 8 levels follow (256 lanes); a join adds once and
    multiplies the side below the maximum by an exponential (2^-22, its argument 1.5 U a distance that is at most the term's own).
    A term passes under a larger maximum at most a few times; 6 are allowed.  Nothing of this grows with the maximum itself."""
    x, w, t, sure = exact_logits(n, vocab, mean, deviation, n + vocab)
    call = Call(gm, dev, F16, x, w, t, mean=0)
    losses, lse, total = call.forward()
    call.close()
    l = torch.from_numpy(x).cuda() @ torch.from_numpy(w).cuda().T
    at = torch.from_numpy(t.astype(np.int64)).cuda()[:, None]
    z = l.gather(1, at)[:, 0].cpu().numpy()
    others = l.scatter(1, at, -np.inf)
    top = others.max(1).values
    e = torch.exp(others - top[:, None])
    distance = torch.where(e > 0, (top[:, None] - others).clamp(max=1e4), torch.zeros_like(e))
    spread = ((e * distance).sum(1) / e.sum(1)).cpu().numpy()
    rest = torch.logsumexp(others, 1).cpu().numpy()
    want_loss = np.logaddexp(0.0, rest - z)
    want_lse = np.logaddexp(rest, z)
    pieces = vocab / 128 + 8
    relative = 2.0 ** -22 * 8 + 1.5 * U * 7 * spread + U * (32 + pieces / 32 + 16)
    # a sure row: the loss is log1p of that sum times an exponential of an exact difference, two and two units
    assert np.all(np.abs(losses - want_loss)[sure] <= (relative + 2.0 ** -21 + U)[sure] * want_loss[sure]), \
        float(np.max((np.abs(losses - want_loss) / want_loss)[sure]))
    # the others: a difference that is exact, a logarithm, one addition, so nothing beyond roundings of the loss itself
    bound = relative + 2.0 ** -21 + 4 * U * (np.abs(want_loss) + 1)
    assert np.all(np.abs(losses - want_loss)[~sure] <= bound[~sure]), float(np.max((np.abs(losses - want_loss) / bound)[~sure]))
    assert np.all(np.abs(lse - want_lse) <= bound + 2 * U * np.abs(want_lse))
    # 8 losses are added in binary32, the others in 64 bits, one rounding
    assert abs(total[0] - want_loss.sum()) <= (np.where(sure, (relative + 2.0 ** -21 + U) * want_loss, bound) + 9 * U * want_loss).sum()


def sure_rows(dtype, n, dim, vocab, odds, offset, seed):
    """Rows whose targets, all different, have probabilities near 1 - 1 / odds; the products of a target's logit are spread
    over all columns, and all logits lie `offset` higher than their differences need."""
    g = np.random.default_rng(seed)
    w = R.rounded(g.standard_normal((vocab, dim)) / np.sqrt(dim), dtype)
    w[:, :16] = 1.0
    t = g.permutation(vocab)[:n].astype(np.int32)
    unit = w[t].copy()
    unit[:, :16] = 0.0
    unit /= (unit ** 2).sum(1, keepdims=True)
    x = unit * (np.log(vocab) + np.log(odds))
    x[:, :16] = offset / 16
    return R.rounded(x, dtype), w, t


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,dim,vocab", [(200, 4096, 600), (64, 8192, 600), (130, 1024, 3000), (33, 600, 2000)])
@pytest.mark.parametrize("odds,offset", [(99.0, 0.0), (999.0, 0.0), (999.0, 8.0), (20000.0, 8.0)])
@pytest.mark.parametrize("which", [1, 2])
def test_gradient_of_a_sure_target(gm, dev, dtype, n, dim, vocab, odds, offset, which):
    """The target's entry of softmax - onehot, -(1 - p), must be right relative to itself, not to 1.  It is formed from the
    target's logit and the log-sum-exp: their difference is off by the rounding of the latter, 2 U |lse| (its own and
    the subtraction's), and 1 - p by the relative errors of the other entries' exponentials: their logits' errors.
    Those: the tensor cores cut a sum at most by 2^-23 of it per 16 products in binary32, forward in parts of at most 2,048
    columns; taken here as (columns of a part / 16 + 32) 2^-23 of the sum of magnitudes over sqrt(columns), the size the partial
    sums of these random products have.  Then two roundings to the type, of S and of the result."""
    x, w, t = sure_rows(dtype, n, dim, vocab, odds, offset, n + dim)
    call = Call(gm, dev, dtype, x, w, t, mean=0)
    losses, lse, _ = call.forward()
    dx, dw = call.backward(which=which)
    call.close()
    X, W = torch.from_numpy(x).cuda(), torch.from_numpy(w).cuda()
    at = torch.from_numpy(t.astype(np.int64)).cuda()
    l = X @ W.T
    p = torch.softmax(l, 1)
    rows = torch.arange(n, device="cuda")
    others = p.clone()
    others[rows, at] = 0.0
    own = -others.sum(1)                                            # the target's entry, without cancellation
    assert float(own.abs().max()) < 0.2 and float(own.abs().min()) > 1e-6
    s = others.clone()
    s[rows, at] = own
    e_logit = (min(dim, 2048) / 16 + 32) * 2.0 ** -23 * ((X.abs() @ W.abs().T).max(1).values / np.sqrt(dim) + l.abs().max(1).values)
    e_others = (4 * e_logit + 2.0 ** -20)[:, None] * others          # its logit's, the target's, the log-sum-exp's, S's logits in one sum
    extra = dim / 16 * 2.0 ** -23 * l.abs().max(1).values[:, None] * others
    e_s = e_others + extra
    e_s[rows, at] = (4 * e_logit + 2.0 ** -20) * own.abs() + 2 * U * torch.logsumexp(l, 1).abs()
    half = R.HALF_STEP[dtype]
    e_s = e_s + (half + (n + vocab + 16) * 2.0 ** -23) * s.abs()
    tiny = R.TINY[dtype] * (2.0 ** -15 if dtype == F16 else 1.0)
    for got, want, bound in ((dw, s.T @ X, e_s.T @ X.abs() + tiny * X.abs().sum(0)), (dx, s @ W, e_s @ W.abs() + tiny * W.abs().sum(0))):
        want, bound = want.cpu().numpy(), bound.cpu().numpy()
        bound = bound + half * (np.abs(want) + bound) + R.TINY[dtype]
        assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / bound))
    # the same without worst cases: a target's own row of dW, which is nearly a multiple of its hidden state, to the
    # roundings of its type and those of the difference
    want = (s.T @ X)[at].cpu().numpy()
    off = np.linalg.norm(dw[t] - want, axis=1) / np.linalg.norm(want, axis=1)
    limit = 2 * half + (4 * e_logit + 2.0 ** -20).cpu().numpy() + (2 * U * torch.logsumexp(l, 1).abs() / own.abs()).cpu().numpy()
    floor = R.TINY[dtype] * np.sqrt(dim) / np.linalg.norm(want, axis=1)      # results below the type's normal numbers
    assert np.all(off <= limit + floor), float(np.max(off / (limit + floor)))
