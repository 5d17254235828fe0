"""The vocabulary loss where a model is sure of itself: statistics of large logits and small losses, each
against 64 bits."""
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
