"""What a product of the vocabulary loss whose bounded wait ran out leaves behind: gradients that no optimizer step takes.
The wait is made to run out by the self-check, on a barrier that nothing arrives at, with a budget of a few milliseconds."""
import ctypes as C

import numpy as np
import pytest

import lm_ref as R
from test_language_model_gpu import Tied
from test_linear_xent_gpu import Call, make

F16, BF16 = 2, 4


def run_out(gm, dev):
    gave_up = C.c_int(0)
    gm.check(gm.lib.gm_selftest_xent_timeout(dev.h, 4_000_000, C.byref(gave_up)))
    assert gave_up.value == 1


class Quiet(Call):
    """A backward pass that leaves the status alone."""

    def gradients(self, which, base=None, dx=True, dw=True):
        L, dev = self.gm.lib, self.dev
        size = L.gm_linear_xent_workspace_bytes(self.h, which)
        ws = dev.alloc(size)
        p_dx = self.put(np.zeros((self.n, self.dim)), self.ldx) if dx else 0
        p_dw = self.put(np.zeros((self.vocab, self.dim)) if base is None else base, self.ldw) if dw else 0
        self.gm.check(L.gm_linear_xent_backward_async(dev.h, self.h, self.x, self.w, self.t, self.lse, 0, 1.0, p_dx, p_dw, int(base is not None), ws, size))
        out = self.get(p_dx, self.n, self.ldx) if dx else None, self.get(p_dw, self.vocab, self.ldw) if dw else None
        for p in (ws, p_dx, p_dw):
            if p:
                dev.free(p)
        return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,dim,vocab", [(3, 16, 40), (140, 40, 600), (300, 200, 2000)])
def test_gradients_are_not_finite_until_the_status_is_read(gm, dev, dtype, n, dim, vocab):
    x, w, t = make(dtype, n, dim, vocab, n, 0.3)
    t[0] = 1
    call = Quiet(gm, dev, dtype, x, w, t)
    call.forward()
    base = R.rounded(np.random.default_rng(2).standard_normal(w.shape), dtype)
    forms = [(1, None, True, True), (2, None, True, True), (2, base, True, True), (1, None, True, False), (1, None, False, True), (1, base, False, True)]
    good = [call.gradients(*f) for f in forms]
    run_out(gm, dev)
    for f in forms:
        dx, dw = call.gradients(*f)
        live = (t >= 0) & (t < vocab)
        assert dx is None or (np.isnan(dx[live]).all() and not dx[~live].any())
        assert dw is None or np.isnan(dw).all()
    assert gm.lib.gm_linear_xent_status(dev.h) == -12
    for f, (want_dx, want_dw) in zip(forms, good):
        dx, dw = call.gradients(*f)
        assert (dx is None or np.array_equal(dx, want_dx)) and (dw is None or np.array_equal(dw, want_dw))
    assert gm.lib.gm_linear_xent_status(dev.h) == 0
    call.close()


@pytest.mark.gpu
def test_the_mixed_step_skips_such_a_gradient(gm, dev):
    """The chain that a trainer queues without looking at the status in between."""
    t = Tied(gm, dev, 150, 48, 400)
    t.step()
    before, st = dev.to_host(t.d_w, 400 * 48), t.state()
    assert st.adam_t == 1 and st.last_overflow == 0
    run_out(gm, dev)
    t.step()
    after = t.state()
    assert after.last_overflow == 1 and after.adam_t == 1 and after.skipped == st.skipped + 1
    assert np.array_equal(dev.to_host(t.d_w, 400 * 48), before)
    assert gm.lib.gm_linear_xent_status(dev.h) == -12
    t.step()
    assert t.state().adam_t == 2 and np.isfinite(dev.to_host(t.d_w, 400 * 48)).all()
    t.close()
