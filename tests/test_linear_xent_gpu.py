"""The vocabulary loss and both gradients against their definition in 64 bits.

Error bounds.  With a = sum |x w| of a logit, a product of D terms summed in binary32 (the tensor
cores may cut instead of round, 2^-23 a step) is off by at most e = (D + 8) 2^-23 a.  A
log-sum-exp adds the two-ulp exponential, the rounded reference (2^-22 of the largest logit) and
sums of at most 256 + V / 2048 steps.  A probability is then off by e + the error of lse,
relatively; S is rounded to the type (half a step); a gradient is a sum of products of those in
binary32 and rounded once more."""
import ctypes as C

import numpy as np
import pytest
import torch

import lm_ref as R

F16, BF16 = 2, 4


def make(dtype, n, dim, vocab, seed, ignored=0.0, gain=1.0):
    g = np.random.default_rng(seed)
    x = R.rounded(gain * g.standard_normal((n, dim)), dtype)
    w = R.rounded(g.standard_normal((vocab, dim)) / np.sqrt(dim), dtype)
    t = g.integers(0, vocab, n).astype(np.int32)
    t[g.random(n) < ignored] = -100
    return x, w, t


def reference(x, w, t, c, base=None):
    """losses, lse, dX, dW (times c), and an error bound for each, without the outputs' own rounding."""
    X, W = torch.from_numpy(x).cuda(), torch.from_numpy(w).cuda()
    n, dim, vocab = X.shape[0], X.shape[1], W.shape[0]
    T = torch.from_numpy(t.astype(np.int64)).cuda()
    ok = (T >= 0) & (T < vocab)
    X = torch.where(ok[:, None], X, torch.zeros_like(X))
    at = torch.where(ok, T, torch.zeros_like(T))
    l = X @ W.T
    lse = torch.logsumexp(l, 1)
    losses = lse - l.gather(1, at[:, None])[:, 0]
    p = torch.exp(l - lse[:, None])
    s = p.clone()
    s[torch.arange(n, device="cuda"), at] -= 1
    s *= ok[:, None]
    p = p * ok[:, None]
    e = (dim + 8) * 2.0 ** -23 * (X.abs() @ W.abs().T).max(1).values
    e_lse = e + 2.0 ** -22 * (l.abs().max(1).values + 16) + (256 + vocab / 2048) * 2.0 ** -24
    e_loss = 2 * e_lse + 2.0 ** -24 * losses.abs()
    zero = torch.zeros_like(lse)
    out = {"losses": torch.where(ok, losses, zero), "lse": torch.where(ok, lse, zero), "dx": c * (s @ W), "dw": c * (s.T @ X)}
    e_p = (e + e_lse + 2.0 ** -20)[:, None]
    err = {"losses": e_loss, "lse": e_lse}
    err["dx_p"], err["dw_p"] = abs(c) * ((p * e_p) @ W.abs()), abs(c) * ((p * e_p).T @ X.abs())
    err["dx_s"], err["dw_s"] = abs(c) * (s.abs() @ W.abs()), abs(c) * (s.abs().T @ X.abs())
    # S below the type's smallest numbers, 2^-15 of them in fp16
    err["dx_t"], err["dw_t"] = abs(c) * (ok[:, None] * W.abs().sum(0)[None, :]), abs(c) * X.abs().sum(0)[None, :].expand(vocab, dim)
    return {k: v.cpu().numpy() for k, v in out.items()}, {k: v.cpu().numpy() for k, v in err.items()}, int(ok.sum())


def grad_bound(err, which, ref, dtype, terms, base=None):
    half = R.HALF_STEP[dtype]
    tiny = R.TINY[dtype] * (2.0 ** -15 if dtype == F16 else 1.0)
    b = 1.01 * (err[which + "_p"] + (half + (terms + 16) * 2.0 ** -23) * err[which + "_s"]) + tiny * err[which + "_t"]
    size = np.abs(ref) + b + (np.abs(base) if base is not None else 0)
    return b + half * size + 2.0 ** -22 * size + R.TINY[dtype]


class Call:
    """Device buffers of one loss and its calls."""

    def __init__(self, gm, dev, dtype, x, w, t, mean=1, ex=0, ew=0, shift=0):
        self.gm, self.dev, self.dtype = gm, dev, dtype
        (self.n, self.dim), self.vocab = x.shape, w.shape[0]
        self.ldx, self.ldw = self.dim + ex, (self.dim + 7) // 8 * 8 + ew
        self.shift = shift
        self.h = gm.LinearXent(dtype=dtype, tokens=self.n, dim=self.dim, vocab=self.vocab, ld_hidden=self.ldx, ld_weight=self.ldw, mean=mean)
        self.x, self.w, self.t = self.put(x, self.ldx, shift), self.put(w, self.ldw), dev.to_device(t)
        self.losses, self.lse, self.total = (dev.to_device(np.full(k, -7.0, np.float32)) for k in (self.n + 4, self.n + 4, 4))
        self.keep = [self.x, self.w, self.t, self.losses, self.lse, self.total]

    def put(self, a, ld, shift=0):
        b = R.bytes_of(R.strided(a, ld, self.dtype), self.dtype)
        return self.dev.to_device(np.concatenate([np.zeros(shift * 2, np.uint8), b, np.zeros(64, np.uint8)]))

    def get(self, p, rows, ld, shift=0):
        raw = self.dev.to_host(p, shift * 2 + rows * ld * 2 + 64, np.uint8)
        assert not raw[:shift * 2].any() and not raw[shift * 2 + rows * ld * 2:].any(), "bytes around the matrix were written"
        v = R.values_of(raw[shift * 2:shift * 2 + rows * ld * 2].copy(), self.dtype).reshape(rows, ld)
        assert np.all(v[:, self.dim:] == -7.0), "columns behind the row were written"
        return v[:, :self.dim]

    def room(self, which):
        size = self.gm.lib.gm_linear_xent_workspace_bytes(self.h, which)
        assert size > 0, self.gm.last_error()
        ws = self.dev.to_device(np.full(size + 256, 0xFF, np.uint8))          # NaN in every type
        return ws, size

    def end_room(self, ws, size):
        assert np.all(self.dev.to_host(ws, size + 256, np.uint8)[size:] == 0xFF), "the workspace was overrun"
        self.dev.free(ws)

    def forward(self):
        ws, size = self.room(0)
        self.gm.check(self.gm.lib.gm_linear_xent_forward_async(self.dev.h, self.h, self.x + self.shift * 2, self.w, self.t, self.losses, self.lse,
                                                               self.total, ws, size), "forward")
        losses, lse, total = (self.dev.to_host(p, k) for p, k in ((self.losses, self.n + 4), (self.lse, self.n + 4), (self.total, 4)))
        self.end_room(ws, size)
        assert np.all(losses[self.n:] == -7) and np.all(lse[self.n:] == -7) and np.all(total[2:] == -7)
        return losses[:self.n], lse[:self.n], total[:2]

    def backward(self, grad_scale=1.0, scale=None, which=1, base=None, dx=True, dw=True):
        ws, size = self.room(which)
        b = np.zeros((self.vocab, self.dim)) if base is None else base
        p_dx = self.put(np.zeros((self.n, self.dim)), self.ldx, self.shift) if dx else 0
        p_dw = self.put(b, self.ldw) if dw else 0
        p_scale = self.dev.to_device(np.array([scale], np.float32)) if scale is not None else 0
        self.gm.check(self.gm.lib.gm_linear_xent_backward_async(self.dev.h, self.h, self.x + self.shift * 2, self.w, self.t, self.lse, p_scale,
                                                                grad_scale, p_dx + self.shift * 2 if dx else 0, p_dw, int(base is not None), ws, size),
                      "backward")
        got_dx = self.get(p_dx, self.n, self.ldx, self.shift) if dx else None
        got_dw = self.get(p_dw, self.vocab, self.ldw) if dw else None
        self.end_room(ws, size)
        assert self.gm.lib.gm_linear_xent_status(self.dev.h) == 0
        for q in (p_dx, p_dw, p_scale):
            if q:
                self.dev.free(q)
        return got_dx, got_dw

    def close(self):
        for p in self.keep:
            self.dev.free(p)


def check_forward(got, ref, err, count, mean):
    losses, lse, total = got
    assert np.all(np.abs(losses - ref["losses"]) <= err["losses"])
    assert np.all(np.abs(lse - ref["lse"]) <= err["lse"])
    assert total[1] == count
    want = ref["losses"].sum() / (max(count, 1) if mean else 1)
    # the losses' own errors, 32-term sums in binary32, one rounding
    bound = (err["losses"] * (ref["losses"] != 0)).sum() / (max(count, 1) if mean else 1) + 34 * 2.0 ** -24 * abs(want)
    assert abs(total[0] - want) <= bound


def check_backward(got, ref, err, call, base=None):
    dx, dw = got
    if dx is not None:
        b = grad_bound(err, "dx", ref["dx"], call.dtype, call.vocab)
        assert np.all(np.abs(dx - ref["dx"]) <= b), float(np.max(np.abs(dx - ref["dx"]) / b))
    if dw is not None:
        want = ref["dw"] + (base if base is not None else 0)
        b = grad_bound(err, "dw", ref["dw"], call.dtype, call.n, base)
        assert np.all(np.abs(dw - want) <= b), float(np.max(np.abs(dw - want) / b))


SIZES = [(1, 8, 1), (1, 1, 7), (3, 40, 255), (130, 64, 256), (257, 100, 257), (300, 520, 1000), (64, 72, 5003), (513, 136, 515), (2, 1024, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,dim,vocab", SIZES)
def test_forward(gm, dev, dtype, n, dim, vocab):
    for ignored, mean, ex, shift in [(0.0, 1, 0, 0), (0.5, 0, 3, 0), (0.3, 1, 8, 1)]:
        x, w, t = make(dtype, n, dim, vocab, n + dim, ignored)
        call = Call(gm, dev, dtype, x, w, t, mean, ex, 8 * (ex > 0), shift)
        ref, err, count = reference(x, w, t, 1.0)
        check_forward(call.forward(), ref, err, count, mean)
        call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,dim,vocab", SIZES)
def test_backward(gm, dev, dtype, n, dim, vocab):
    for ignored, mean, ex, shift, which, scale in [(0.0, 1, 0, 0, 1, None), (0.5, 0, 3, 0, 2, 4.0), (0.3, 1, 8, 1, 2, 1024.0)]:
        x, w, t = make(dtype, n, dim, vocab, n + dim, ignored)
        call = Call(gm, dev, dtype, x, w, t, mean, ex, 8 * (ex > 0), shift)
        count = int(np.sum((t >= 0) & (t < vocab)))
        c = 0.5 * (scale or 1.0) / (max(count, 1) if mean else 1)
        ref, err, _ = reference(x, w, t, c)
        call.forward()
        check_backward(call.backward(0.5, scale, which), ref, err, call)
        base = R.rounded(np.random.default_rng(5).standard_normal(w.shape), dtype)
        check_backward(call.backward(0.5, scale, which, base), ref, err, call, base)
        call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_one_gradient_at_a_time_and_twice_the_same_bits(gm, dev, dtype):
    x, w, t = make(dtype, 200, 96, 700, 9, 0.2)
    call = Call(gm, dev, dtype, x, w, t)
    a = call.forward()
    b = call.forward()
    assert all(np.array_equal(p, q) for p, q in zip(a, b))
    both = call.backward(which=2)
    only_x, only_w = call.backward(which=2, dw=False), call.backward(which=2, dx=False)
    assert np.array_equal(both[0], only_x[0]) and np.array_equal(both[1], only_w[1])
    again = call.backward(which=2)
    assert np.array_equal(both[0], again[0]) and np.array_equal(both[1], again[1])
    call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_without_a_target_may_hold_anything(gm, dev, dtype):
    """NaN and infinities in padded rows reach neither the loss nor a gradient; targets on either side of the table."""
    x, w, t = make(dtype, 150, 64, 300, 2)
    t[::3], t[1] = -1, 300
    clean = Call(gm, dev, dtype, x, w, t)
    want_f, want_b = clean.forward(), clean.backward()
    bad = x.copy()
    bad[::3], bad[1] = np.nan, np.inf
    call = Call(gm, dev, dtype, bad, w, t)
    got_f, got_b = call.forward(), call.backward()
    for a, b in zip(list(want_f) + list(want_b), list(got_f) + list(got_b)):
        assert np.array_equal(a, b)
    assert np.all(got_b[0][::3] == 0) and np.all(got_f[0][::3] == 0)
    clean.close()
    call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("mean", [0, 1])
def test_no_row_with_a_target(gm, dev, mean):
    x, w, t = make(F16, 70, 24, 90, 3)
    t[:] = -100
    call = Call(gm, dev, F16, x, w, t, mean)
    losses, lse, total = call.forward()
    assert not losses.any() and not lse.any() and total[0] == 0 and total[1] == 0
    dx, dw = call.backward()
    assert not dx.any() and not dw.any()
    base = R.rounded(np.random.default_rng(0).standard_normal(w.shape), F16)
    assert np.array_equal(call.backward(base=base)[1], base)
    call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_logits(gm, dev, dtype):
    """Logits of several hundred: the exponentials neither overflow nor lose the row."""
    x, w, t = make(dtype, 140, 64, 600, 4, gain=60.0)
    call = Call(gm, dev, dtype, x, w, t)
    ref, err, count = reference(x, w, t, 1.0 / 140)
    assert np.abs(ref["lse"]).max() > 150
    check_forward(call.forward(), ref, err, count, 1)
    check_backward(call.backward(which=2), ref, err, call)
    call.close()


@pytest.mark.gpu
def test_nan_reaches_its_row_and_an_infinite_gradient_is_infinite(gm, dev):
    """What the overflow check of the mixed-precision step looks for arrives in the gradient."""
    x, w, t = make(F16, 20, 16, 40, 6)
    x[3, 5] = np.nan
    call = Call(gm, dev, F16, x, w, t)
    losses, lse, total = call.forward()
    assert np.isnan(losses[3]) and np.isnan(total[0]) and np.isfinite(np.delete(losses, 3)).all()
    dx, dw = call.backward()
    assert np.isnan(dx[3]).all() and np.isfinite(np.delete(dx, 3, 0)).all() and np.isnan(dw).all()
    call.close()
    x, w, t = make(F16, 20, 16, 40, 6)
    call = Call(gm, dev, F16, x, w, t)
    call.forward()
    assert np.isinf(call.backward(scale=1e9)[1]).any()
    call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [20, 140])
def test_infinite_logits(gm, dev, n):
    """Entries masked by -inf: as targets they have an infinite loss, and their rows' log-sum-exp and gradient are
    those of the other entries.  A target with logit +inf has no loss: NaN, in the total too."""
    x, w, t = make(F16, n, 24, 300, 16)
    x[:, -1], w[:, -1] = 1.0, 0.0
    masked = np.arange(300) % 7 == 3
    t[::5] = 3
    left = np.flatnonzero(~masked)
    fake = np.where(masked[t], 0, np.searchsorted(left, t)).astype(np.int32)       # the table without the masked entries
    ref, err, _ = reference(x, w[left], fake, 1.0)
    w[masked, -1] = -np.inf
    call = Call(gm, dev, F16, x, w, t, mean=0)
    losses, lse, total = call.forward()
    hit = masked[t]
    assert hit.any() and np.all(losses[hit] == np.inf) and total[0] == np.inf and total[1] == n
    assert np.all(np.abs(losses[~hit] - ref["losses"][~hit]) <= err["losses"][~hit])
    assert np.all(np.abs(lse - ref["lse"]) <= err["lse"])
    dw = call.backward(dx=False)[1]
    l = np.where(masked[None, :], -np.inf, x @ np.where(np.isinf(w), 0, w).T)
    s = np.exp(l - np.logaddexp.reduce(l, 1)[:, None])
    s[np.arange(n), t] -= 1
    want = s.T @ x
    err["dw_s"] = (np.abs(s).T @ np.abs(x))[left]
    assert np.all(np.abs(dw - want)[left] <= grad_bound(err, "dw", want[left], F16, n))
    whole = -np.stack([x[t == v].sum(0) for v in np.flatnonzero(masked)])           # softmax is 0 there
    size = np.stack([np.abs(x[t == v]).sum(0) for v in np.flatnonzero(masked)])
    assert np.all(np.abs(dw[masked] - whole) <= 1.01 * R.HALF_STEP[F16] * np.abs(whole) + (n + 2) * 2.0 ** -23 * size)
    call.close()
    w[masked, -1] = 0.0
    w[3, -1] = np.inf
    call = Call(gm, dev, F16, x, w, t)
    losses, lse, total = call.forward()
    assert np.isnan(losses[t == 3]).all() and not np.isfinite(losses).any() and np.isnan(total[0])
    call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [64, 192])
def test_long_sums_do_not_shift_the_loss(gm, dev, n):
    """The tensor cores cut where they add, 16 products at a time: half a unit in the last place on average, at most 2^-24 of
    the sum so far, always towards zero.  The forward pass takes 8,192 columns in six sums, so a mean loss is off by at most
    2^-24 of the sums so far of those, weighted with the probabilities (rounding errors average out over rows and entries); in
    one sum it would be off by about twice that bound."""
    x, w, t = make(BF16, n, 8192, 640, 33)
    w = R.rounded(w * (0.02 * np.sqrt(8192)), BF16)
    call = Call(gm, dev, BF16, x, w, t)
    total = call.forward()[2][0]
    call.close()
    X, W = torch.from_numpy(x).cuda().view(n, 512, 16), torch.from_numpy(w).cuda().view(640, 512, 16)
    steps = torch.einsum("nsk,vsk->snv", X, W)
    l = steps.sum(0)
    ends = [4 * (128 * c // 6) for c in range(7)]                     # a block of 64 columns is four steps
    so_far = sum(steps[a:b].cumsum(0).abs().sum(0) for a, b in zip(ends, ends[1:]))
    p = torch.softmax(l, 1)
    want = float(torch.nn.functional.cross_entropy(l, torch.from_numpy(t.astype(np.int64)).cuda()))
    bound = float((p * so_far).sum(1).mean()) * 2.0 ** -24
    assert abs(total - want) <= bound + 2.0 ** -22 * want


@pytest.mark.gpu
def test_gradient_against_differences(gm, dev):
    """The summed loss along a direction: a central difference of the library's own forward pass, whose
    step leaves at most h^2 of third derivatives (bounded by |d|^3) and 2 error(total) / h of rounding."""
    x, w, t = make(BF16, 24, 32, 100, 8, 0.2)
    g = np.random.default_rng(1)
    step = 2.0 ** -7
    dirn = R.rounded(np.sign(g.standard_normal(w.shape)) * step, BF16)
    w = R.rounded(np.round(w * 8) / 8, BF16)                       # w +- step is exact in bf16
    totals = []
    for s in (1, -1):
        call = Call(gm, dev, BF16, x, w + s * dirn, t, mean=0)
        totals.append(float(call.forward()[2][0]))
        call.close()
    call = Call(gm, dev, BF16, x, w, t, mean=0)
    call.forward()
    dw = call.backward()[1]
    ref, err, _ = reference(x, w, t, 1.0)
    third = (np.abs(x).sum(1) * step) ** 3                        # |third derivative of lse along d| <= 2 max|d.x|^3 and more
    bound = third.sum() / 3 + 2 * err["losses"].sum() + (grad_bound(err, "dw", ref["dw"], BF16, 24) * np.abs(dirn)).sum()
    assert abs((totals[0] - totals[1]) / 2 - np.sum(dw * dirn)) <= bound
    call.close()


@pytest.mark.gpu
def test_captured_forward_and_backward_replay_on_new_inputs(gm, dev):
    """One graph of both passes, replayed after the inputs changed, against eager calls."""
    n, dim, vocab = 300, 64, 900
    L = gm.lib
    x, w, t = make(F16, n, dim, vocab, 10, 0.1)
    x2, w2, t2 = make(F16, n, dim, vocab, 11, 0.6)
    call = Call(gm, dev, F16, x, w, t)
    size = L.gm_linear_xent_workspace_bytes(call.h, 1)
    ws, dx, dw = dev.alloc(size), dev.alloc(n * dim * 2), dev.alloc(vocab * dim * 2)

    def both():
        gm.check(L.gm_linear_xent_forward_async(dev.h, call.h, call.x, call.w, call.t, call.losses, call.lse, call.total, ws, size))
        gm.check(L.gm_linear_xent_backward_async(dev.h, call.h, call.x, call.w, call.t, call.lse, 0, 1.0, dx, dw, 0, ws, size))

    def results():
        return [dev.to_host(p, k, np.uint8) for p, k in ((call.losses, n * 4), (call.lse, n * 4), (call.total, 8), (dx, n * dim * 2), (dw, vocab * dim * 2))]
    both()
    dev.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(L.gm_device_stream(dev.h))):
        both()
    for a, b, c in ((x, w, t), (x2, w2, t2), (x, w, t)):
        dev.upload(call.x, R.bytes_of(a, F16))
        dev.upload(call.w, R.bytes_of(b, F16))
        dev.upload(call.t, c)
        both()
        want = results()
        for p, k in ((call.losses, n * 4), (dx, n * dim * 2), (dw, vocab * dim * 2)):
            gm.check(L.gm_buffer_zero(dev.h, p, k))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(np.array_equal(p, q) for p, q in zip(want, results()))
    del g
    for p in (ws, dx, dw):
        dev.free(p)
    call.close()


@pytest.mark.gpu
def test_a_wait_that_runs_out_is_reported_and_the_device_stays_usable(gm, dev):
    """The bounded wait of the products, on a barrier that nothing arrives at, with a budget of a few
    milliseconds; what follows is what a product that gave up would leave."""
    L = gm.lib
    x, w, t = make(F16, 140, 32, 300, 1)
    call = Call(gm, dev, F16, x, w, t)
    good = call.forward()
    gave_up = C.c_int(0)
    assert L.gm_linear_xent_status(dev.h) == 0
    gm.check(L.gm_selftest_xent_timeout(dev.h, 4_000_000, C.byref(gave_up)))
    assert gave_up.value == 1
    assert np.isnan(call.forward()[2][0])
    assert L.gm_linear_xent_status(dev.h) == -12 and "ran out" in gm.last_error()
    assert L.gm_linear_xent_status(dev.h) == 0
    assert all(np.array_equal(a, b) for a, b in zip(good, call.forward()))
    assert L.gm_selftest_xent_timeout(dev.h, 0, C.byref(gave_up)) == -10 and L.gm_selftest_xent_timeout(dev.h, 1, None) == -10
    call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 64, 65, 127, 128, 129, 1024, 1025, 2048, 2049])
def test_every_form_of_the_forward_pass(gm, dev, dtype, n):
    """Around the row counts where another form takes over, with hidden states that can and cannot be read in place."""
    for vocab, ex, shift in [(1000, 0, 0), (37, 3, 0), (5000, 8, 1)]:
        x, w, t = make(dtype, n, 72, vocab, n + vocab, 0.3 if n > 1 else 0.0)
        call = Call(gm, dev, dtype, x, w, t, 1, ex, 0, shift)
        ref, err, count = reference(x, w, t, 1.0)
        check_forward(call.forward(), ref, err, count, 1)
        call.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n,dim,vocab", [(700, 1300, 2000), (5000, 300, 700), (256, 2048, 257), (1000, 600, 9000)])
def test_shares_of_k_and_pieces(gm, dev, n, dim, vocab):
    """Sizes whose dX has whole rounds of tiles, a split last round, or nothing but split tiles, in one
    piece of the vocabulary and in many."""
    x, w, t = make(BF16, n, dim, vocab, 5, 0.1)
    call = Call(gm, dev, BF16, x, w, t)
    count = int((t >= 0).sum())
    ref, err, _ = reference(x, w, t, 1.0 / count)
    call.forward()
    for which in (1, 2):
        check_backward(call.backward(which=which), ref, err, call)
    call.close()


@pytest.mark.gpu
def test_table_gradient_at_an_odd_address(gm, dev):
    """dW needs no alignment beyond its type's, with and without accumulation."""
    L = gm.lib
    x, w, t = make(F16, 90, 40, 300, 12)
    call = Call(gm, dev, F16, x, w, t)
    call.forward()
    want = call.backward(dx=False)[1]
    base = R.rounded(np.random.default_rng(3).standard_normal(w.shape), F16)
    ws, size = call.room(1)
    for add in (0, 1):
        raw = np.concatenate([np.zeros(2, np.uint8), R.bytes_of(base, F16), np.zeros(62, np.uint8)])
        p = dev.to_device(raw)
        gm.check(L.gm_linear_xent_backward_async(dev.h, call.h, call.x, call.w, call.t, call.lse, 0, 1.0, 0, p + 2, add, ws, size))
        got = dev.to_host(p, raw.size, np.uint8)
        v = R.values_of(got[2:2 + base.size * 2].copy(), F16).reshape(base.shape)
        if add:
            assert np.all(np.abs(v - (base + want)) <= R.HALF_STEP[F16] * (np.abs(base + want) + np.abs(want) * 1.01) + 2 * R.TINY[F16])
        else:
            assert np.array_equal(v, want)
        assert not got[:2].any() and not got[2 + base.size * 2:].any()
        dev.free(p)
    call.end_room(ws, size)
    call.close()


@pytest.mark.gpu
def test_refusals(gm, dev):
    L = gm.lib
    n, dim, vocab = 4, 16, 32

    def loss(dtype=F16, tokens=n, dim=dim, vocab=vocab, ld_hidden=16, ld_weight=16):
        return gm.LinearXent(dtype=dtype, tokens=tokens, dim=dim, vocab=vocab, ld_hidden=ld_hidden, ld_weight=ld_weight, mean=1)
    ok = loss()
    size = L.gm_linear_xent_workspace_bytes(ok, 1)
    least = L.gm_linear_xent_workspace_bytes(ok, 2)
    x, w, t, losses, lse, total, ws = (dev.alloc(k) for k in (n * dim * 2, vocab * dim * 2, n * 4, n * 4, n * 4, 8, size))
    dx, dw = dev.alloc(n * dim * 2), dev.alloc(vocab * dim * 2)
    before = L.gm_device_launch_count(dev.h)

    def fwd(rc, h=ok, x=x, w=w, t=t, losses=losses, lse=lse, total=total, ws=ws, size=size, d=None):
        assert L.gm_linear_xent_forward_async(dev.h if d is None else d, h, x, w, t, losses, lse, total, ws, size) == rc, gm.last_error()

    def bwd(rc, h=ok, x=x, w=w, t=t, lse=lse, scale=0, dx=dx, dw=dw, ws=ws, size=size, d=None):
        assert L.gm_linear_xent_backward_async(dev.h if d is None else d, h, x, w, t, lse, scale, 1.0, dx, dw, 0, ws, size) == rc, gm.last_error()
    for call in (fwd, bwd):
        call(-1, d=0)
        call(-10, h=None)
        for bad in (loss(dtype=0), loss(dtype=3), loss(ld_hidden=15), loss(ld_weight=15), loss(ld_weight=20)):
            call(-10, h=bad)
        for bad in (loss(tokens=0), loss(dim=0), loss(vocab=0), loss(tokens=-5), loss(tokens=1 << 29), loss(vocab=1 << 29), loss(tokens=1 << 28, vocab=1 << 28),
                    loss(tokens=n + 1), loss(vocab=vocab + 1)):
            call(-9, h=bad)
        call(-4, x=0)
        call(-4, w=0)
        call(-4, t=0)
        call(-4, lse=0)
        call(-4, ws=0)
        call(-10, ws=ws + 16)
        call(-10, x=x + 1)
        call(-10, w=w + 2)
        call(-9, size=least - 1 if call is bwd else L.gm_linear_xent_workspace_bytes(ok, 0) - 1)
    fwd(-4, losses=0)
    fwd(-4, total=0)
    bwd(-4, dx=0, dw=0)
    bwd(-10, scale=total + 2)
    bwd(-9, dx=total)
    bwd(-9, dw=total)
    assert L.gm_device_launch_count(dev.h) == before
    assert L.gm_linear_xent_status(0) == -1 and L.gm_linear_xent_status(dev.h) == 0
    for p in (x, w, t, losses, lse, total, ws, dx, dw):
        dev.free(p)


def test_workspace_sizes_need_no_device(gm):
    L = gm.lib
    h = gm.LinearXent(dtype=F16, tokens=100, dim=64, vocab=100000, ld_hidden=64, ld_weight=64, mean=1)
    f, r, s = (L.gm_linear_xent_workspace_bytes(h, k) for k in (0, 1, 2))
    assert 0 < s <= r and f <= r
    assert L.gm_linear_xent_workspace_bytes(h, 3) == -1 and L.gm_linear_xent_workspace_bytes(None, 0) == -1
    h.ld_weight = 68
    assert L.gm_linear_xent_workspace_bytes(h, 0) == -1
