"""Vocabulary entries masked by the type's lowest number, as others mask by -inf: through a column of the table that all hidden
states hold a one in.  Whole tiles, halves of them and single entries are masked."""
import numpy as np
import pytest
import torch

import lm_ref as R
from test_linear_xent_gpu import Call, grad_bound, make, reference

F16, BF16 = 2, 4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [1, 20, 50, 100, 140, 300])
@pytest.mark.parametrize("masked", [[(256, 512)], [(0, 128), (640, 700)], [(0, 600)], [(5, 6), (128, 256), (301, 333)]])
@pytest.mark.parametrize("dim", [24, 2072])
def test_masked_by_the_lowest_number(gm, dev, dtype, n, masked, dim):
    """Their probabilities are exactly 0: losses, log-sum-exps and gradients are those of the other entries, within the bounds
    of the definition over these (fp16's lowest number is a logit like others, and 65,000 below them).  The bound of a logit is
    that of the other columns: the ones' column adds a zero to an unmasked logit."""
    vocab = 700
    hidden = np.zeros(vocab, bool)
    for a, b in masked:
        hidden[a:b] = True
    left = np.flatnonzero(~hidden)
    x, w, _ = make(dtype, n, dim, vocab, n + dim)
    x[:, -1], w[:, -1] = 1.0, 0.0
    fake = np.random.default_rng(n).integers(0, len(left), n).astype(np.int32)
    ref, err, _ = reference(x, w[left], fake, 1.0)
    w[hidden, -1] = float(torch.finfo(R.TORCH[dtype]).min)
    call = Call(gm, dev, dtype, x, w, left[fake].astype(np.int32), mean=0)
    losses, lse, total = call.forward()
    assert np.all(np.abs(losses - ref["losses"]) <= err["losses"]) and np.all(np.abs(lse - ref["lse"]) <= err["lse"])
    assert np.isfinite(total).all()
    for which in (1, 2):
        dx, dw = call.backward(which=which)
        assert not dw[hidden].any()
        assert np.all(np.abs(dw[left] - ref["dw"]) <= grad_bound(err, "dw", ref["dw"], dtype, n))
        assert np.all(np.abs(dx - ref["dx"]) <= grad_bound(err, "dx", ref["dx"], dtype, vocab))
    call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [20, 140])
def test_a_row_of_nothing_but_the_lowest_number(gm, dev, n):
    """All its logits are one and the same: the loss is log of the vocabulary, the log-sum-exp that number."""
    vocab, dim = 700, 24
    x, w, t = make(BF16, n, dim, vocab, 3)
    x[:, -1], w[:, -1] = 0.0, float(torch.finfo(torch.bfloat16).min)
    want = Call(gm, dev, BF16, x, w, t, mean=0)
    good = want.forward()[0]
    want.close()
    x[::2] = 0.0
    x[::2, -1] = 1.0
    call = Call(gm, dev, BF16, x, w, t, mean=0)
    losses, lse, _ = call.forward()
    call.close()
    assert np.all(np.abs(losses[::2] - np.log(vocab)) <= 2.0 ** -20 * np.log(vocab))
    assert np.all(lse[::2] == np.float32(torch.finfo(torch.bfloat16).min))
    assert np.array_equal(losses[1::2], good[1::2])
