"""Calls of the language-model operators that the header allows and no other test makes."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import lm_ref as R
from test_linear_xent_gpu import Call, check_backward, check_forward, make, reference

F32, F16, BF16 = 0, 2, 4


def P(t):
    return t.data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [7, 33, 100, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_few_rows_without_a_target_may_hold_anything(gm, dev, n, dtype):
    """Up to 128 rows are read in place, those without a target too; NaN and infinities in them reach nothing."""
    x, w, t = make(dtype, n, 72, 1001, n)
    t[::3], t[1] = -1, 1001
    bad = x.copy()
    bad[::3], bad[1, :9] = np.nan, np.inf
    for ex, shift in ((0, 0), (3, 1)):
        clean, dirty = Call(gm, dev, dtype, x, w, t, 1, ex, 0, shift), Call(gm, dev, dtype, bad, w, t, 1, ex, 0, shift)
        for a, b in zip(list(clean.forward()) + list(clean.backward()), list(dirty.forward()) + list(dirty.backward())):
            assert np.isfinite(b).all() and np.array_equal(a, b)
        clean.close()
        dirty.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 30, 140])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_vocabulary_of_one(gm, dev, n, dtype):
    """The only entry has probability 1: losses and gradients are exactly 0, the log-sum-exp is the logit."""
    x, w, t = make(dtype, n, 200, 1, n)
    call = Call(gm, dev, dtype, x, w, t)
    losses, lse, total = call.forward()
    assert not losses.any() and total[0] == 0 and total[1] == n
    assert np.all(np.abs(lse - (x @ w.T)[:, 0]) <= (200 / 128 + 9) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T)[:, 0])
    for which in (1, 2):
        dx, dw = call.backward(which=which)
        assert not dx.any() and not dw.any()
    call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 300])
def test_all_rows_with_one_target_and_a_target_at_every_border(gm, dev, n):
    """The same entry again and again, and entries around the borders of warps, halves of tiles, tiles and pieces."""
    for vocab, targets in ((700, [511]), (700, [0, 31, 32, 127, 128, 255, 256, 383, 384, 511, 512, 639, 640, 699])):
        x, w, t = make(F16, n, 40, vocab, n)
        t[:] = np.resize(targets, n)
        call = Call(gm, dev, F16, x, w, t, mean=0)
        ref, err, count = reference(x, w, t, 1.0)
        check_forward(call.forward(), ref, err, count, 0)
        for which in (1, 2):
            check_backward(call.backward(which=which), ref, err, call)
        call.close()


@pytest.mark.gpu
def test_gradients_over_given_statistics(gm, dev):
    """A backward pass with the log-sum-exp of another one's forward pass, here the definition's, rounded: the header asks for the values,
    not for the call.  p is off by twice the rounding of the log-sum-exp more."""
    x, w, t = make(F16, 260, 136, 900, 5, 0.2)
    call = Call(gm, dev, F16, x, w, t, mean=0)
    ref, err, _ = reference(x, w, t, 1.0)
    dev.upload(call.lse, np.concatenate([ref["lse"], np.full(4, -7.0)]).astype(np.float32))
    check_backward(call.backward(), ref, err, call)
    call.close()


@pytest.mark.gpu
def test_between_operations_of_another_stream(gm, dev):
    """The handle's stream and the default stream order each other: inputs that torch writes just before a call
    and outputs that it reads just after, without a wait in between, while the calls' own kernels start early."""
    L = gm.lib
    n, dim, vocab = 96, 512, 3000
    g = torch.Generator(device="cuda").manual_seed(3)
    w = (torch.randn(vocab, dim, generator=g, device="cuda") / 20).half()
    pool = torch.randn(8, n, dim, generator=g, device="cuda").half()
    goals = torch.randint(0, vocab, (8, n), generator=g, device="cuda", dtype=torch.int32)
    slow = torch.randn(4096, 4096, generator=g, device="cuda")
    h = gm.LinearXent(dtype=F16, tokens=n, dim=dim, vocab=vocab, ld_hidden=dim, ld_weight=dim, mean=1)
    e = gm.Embedding(dtype=F16, tokens=n, dim=dim, vocab=vocab, ld_table=dim, ld_out=dim, padding_token=-1, scale=1.0)
    room = torch.empty(max(L.gm_linear_xent_workspace_bytes(h, 1), L.gm_embedding_workspace_bytes(e)), dtype=torch.uint8, device="cuda")
    x, t, y = torch.empty_like(pool[0]), torch.empty_like(goals[0]), torch.empty_like(pool[0])
    losses, lse, total = (torch.empty(k, device="cuda") for k in (n, n, 2))
    dx, dw = torch.empty_like(x), torch.empty_like(w)

    def go(k, wait):
        if not wait:
            torch.mm(slow, slow)
        x.copy_(pool[k])
        t.copy_(goals[k])
        if wait:
            torch.cuda.synchronize()
        gm.check(L.gm_dropout_async(dev.h, F16, n, dim, P(x), dim, 0, 0, P(y), dim, gm.dropout(0.1, 3, k)))
        gm.check(L.gm_linear_xent_forward_async(dev.h, h, P(y), P(w), P(t), P(losses), P(lse), P(total), P(room), room.numel()))
        gm.check(L.gm_linear_xent_backward_async(dev.h, h, P(y), P(w), P(t), P(lse), 0, 64.0, P(dx), P(dw), 0, P(room), room.numel()))
        gm.check(L.gm_embedding_backward_async(dev.h, e, P(t), P(dx), None, P(dw), F16, 1, P(room), room.numel()))
        if wait:
            torch.cuda.synchronize()
        out = [v.clone() for v in (losses, lse, total, dx, dw)]
        for v in (x, y, losses, lse, total, dx, dw):
            v.fill_(0.5)
        t.fill_(1)
        return out
    want = [go(k, True) for k in range(8)]
    got = [go(k, False) for k in list(range(8)) * 3]
    torch.cuda.synchronize()
    for k, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[k % 8]))
    assert L.gm_linear_xent_status(dev.h) == 0


COLD = """
import sys, torch
import gometal_cuda as gm
n, dim, vocab = int(sys.argv[1]), 64, 500
L, P = gm.lib, lambda t: t.data_ptr()
torch.zeros(1, device="cuda")
dev = gm.Device(0)
x, w = torch.randn(n, dim, device="cuda").half(), (torch.randn(vocab, dim, device="cuda") / 8).half()
t = torch.randint(0, vocab, (n,), device="cuda", dtype=torch.int32)
h = gm.LinearXent(dtype=2, tokens=n, dim=dim, vocab=vocab, ld_hidden=dim, ld_weight=dim, mean=1)
e = gm.Embedding(dtype=2, tokens=n, dim=dim, vocab=vocab, ld_table=dim, ld_out=dim, padding_token=-1, scale=1.0)
room = torch.empty(max(L.gm_linear_xent_workspace_bytes(h, 1), L.gm_embedding_workspace_bytes(e)), dtype=torch.uint8, device="cuda")
losses, lse, total = (torch.zeros(k, device="cuda") for k in (n, n, 2))
y, dx, dw = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w)

def go():
    gm.check(L.gm_dropout_async(dev.h, 2, n, dim, P(x), dim, 0, 0, P(y), dim, gm.dropout(0.1, 3)))
    gm.check(L.gm_linear_xent_forward_async(dev.h, h, P(y), P(w), P(t), P(losses), P(lse), P(total), P(room), room.numel()))
    gm.check(L.gm_linear_xent_backward_async(dev.h, h, P(y), P(w), P(t), P(lse), 0, 64.0, P(dx), P(dw), 0, P(room), room.numel()))
    gm.check(L.gm_embedding_backward_async(dev.h, e, P(t), P(dx), None, P(dw), 2, 1, P(room), room.numel()))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(L.gm_device_stream(dev.h))):
    go()
g.replay()
torch.cuda.synchronize()
got = [v.clone() for v in (losses, total, dx, dw)]
go()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, (losses, total, dx, dw))) and float(total[0]) > 0
assert L.gm_linear_xent_status(dev.h) == 0
del g
dev.close()
print("captured cold")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("n", [20, 300])
def test_the_first_call_of_a_process_may_be_captured(gm, n):
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.path.join(os.path.dirname(here), "go-metal_b200", "python"))
    run = subprocess.run([sys.executable, "-c", COLD, str(n)], env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured cold" in run.stdout, run.stderr[-2000:]
