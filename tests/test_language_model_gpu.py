"""The two ends of a tied language model and the mixed-precision step in one run, as a trainer would
chain them on the device's stream: lookup with dropout, vocabulary loss, both gradients into the one
fp16 gradient of the table, and the Adam step that checks, unscales and applies it."""
import ctypes as C

import numpy as np
import pytest
import torch

import lm_ref as R
from test_linear_xent_gpu import grad_bound, reference

F16 = 2


class Tied:
    """A bigram model: the hidden state of a token is its dropped-out embedding, the table is also the head."""

    def __init__(self, gm, dev, n, dim, vocab, scale0=None, p=0.25):
        self.gm, self.dev, self.n, self.dim, self.vocab, self.p = gm, dev, n, dim, vocab, p
        L = gm.lib
        g = np.random.default_rng(n)
        self.master = (g.standard_normal((vocab, dim)) / np.sqrt(dim)).astype(np.float32)
        self.tok = g.integers(0, vocab, n).astype(np.int32)
        self.goal = np.where(g.random(n) < 0.2, -100, g.integers(0, vocab, n)).astype(np.int32)
        size = vocab * dim
        self.d_w, self.d_m, self.d_v = dev.to_device(self.master), dev.to_device(np.zeros(size, np.float32)), dev.to_device(np.zeros(size, np.float32))
        self.d_p = dev.to_device(R.bytes_of(self.master, F16))
        self.d_g, self.d_h, self.d_dh = dev.alloc(size * 2), dev.alloc(n * dim * 2), dev.alloc(n * dim * 2)
        self.d_tok, self.d_goal = dev.to_device(self.tok), dev.to_device(self.goal)
        self.d_losses, self.d_lse, self.d_total = dev.alloc(n * 4), dev.alloc(n * 4), dev.alloc(8)
        self.e = gm.Embedding(dtype=F16, tokens=n, dim=dim, vocab=vocab, ld_table=dim, ld_out=dim, padding_token=-1, scale=2.0)
        self.x = gm.LinearXent(dtype=F16, tokens=n, dim=dim, vocab=vocab, ld_hidden=dim, ld_weight=dim, mean=1)
        self.room = max(L.gm_embedding_workspace_bytes(self.e), L.gm_linear_xent_workspace_bytes(self.x, 1))
        self.d_room = dev.alloc(self.room)
        self.list = dev.tensor_list([[self.d_g], [self.d_w], [self.d_m], [self.d_v], [self.d_p]], [size], [2, 4, 4, 4, 2])
        start = gm.LossScale(scale=scale0, growth=2.0, backoff=0.5, max_scale=2.0 ** 24, interval=2000) if scale0 else None
        self.mixed = L.gm_mixed_create(dev.h, C.byref(start) if start else None, 0.9, 0.999, 0)
        assert self.mixed, gm.last_error()

    def drop(self):
        return self.gm.dropout(self.p, 5, 9)

    def step(self):
        gm, L, h = self.gm, self.gm.lib, self.dev.h
        gm.check(L.gm_embedding_forward_async(h, self.e, self.d_p, self.d_tok, self.d_h, self.drop()))
        gm.check(L.gm_linear_xent_forward_async(h, self.x, self.d_h, self.d_p, self.d_goal, self.d_losses, self.d_lse, self.d_total, self.d_room, self.room))
        gm.check(L.gm_linear_xent_backward_async(h, self.x, self.d_h, self.d_p, self.d_goal, self.d_lse, L.gm_mixed_state_device_ptr(self.mixed), 1.0,
                                                 self.d_dh, self.d_g, 0, self.d_room, self.room))
        gm.check(L.gm_embedding_backward_async(h, self.e, self.d_tok, self.d_dh, self.drop(), self.d_g, F16, 1, self.d_room, self.room))
        gm.check(L.gm_mixed_step_async(h, self.mixed, self.list, 1e-3, 1e-8, 0.0))

    def state(self):
        st = self.gm.LossScale()
        self.gm.check(self.gm.lib.gm_mixed_get_state(self.dev.h, self.mixed, C.byref(st)))
        return st

    def get(self, p, shape, dtype=F16):
        n = int(np.prod(shape)) * R.eb(dtype)
        return R.values_of(self.dev.to_host(p, n, np.uint8), dtype).reshape(shape)

    def close(self):
        self.gm.lib.gm_mixed_destroy(self.mixed)
        self.gm.lib.gm_tensor_list_destroy(self.list)
        for k, p in vars(self).items():
            if k.startswith("d_"):
                self.dev.free(p)


@pytest.mark.gpu
@pytest.mark.parametrize("n,dim,vocab", [(200, 64, 300), (77, 40, 1000), (300, 136, 257)])
def test_gradients_and_step(gm, dev, oracle, n, dim, vocab):
    t = Tied(gm, dev, n, dim, vocab)
    before = t.get(t.d_p, (vocab, dim))
    scale = t.state().scale
    t.step()
    hidden, dh, grad = t.get(t.d_h, (n, dim)), t.get(t.d_dh, (n, dim)), t.get(t.d_g, (vocab, dim))
    keep, up = R.keep_mask(n * dim, t.p, 5, 9)
    keep = keep.reshape(n, dim)
    factor = np.float32(2.0) * up
    want = np.where(keep, before[t.tok].astype(np.float32) * factor, np.float32(0))
    assert np.array_equal(hidden, R.rounded(want, F16))
    # the loss and the head's gradient from the hidden states that were really there
    count = int((t.goal >= 0).sum())
    ref, err, _ = reference(hidden, before, t.goal, scale / count)
    total = t.get(t.d_total, (2,), 0)
    assert total[1] == count and abs(total[0] - ref["losses"].sum() / count) <= err["losses"].mean() + 34 * 2.0 ** -24 * abs(total[0])
    assert np.all(np.abs(dh - ref["dx"]) <= grad_bound(err, "dx", ref["dx"], F16, vocab))
    # both gradients of the table: the head's (rounded once), the lookup's on top (rounded once more);
    # a row takes at most n additions in binary32
    lookup, size = np.zeros((vocab, dim)), np.zeros((vocab, dim))
    np.add.at(lookup, t.tok, np.where(keep, dh, 0.0) * float(factor))
    np.add.at(size, t.tok, np.where(keep, np.abs(dh), 0.0) * float(factor))
    whole = ref["dw"] + lookup
    bound = grad_bound(err, "dw", ref["dw"], F16, n) + (n + 8) * 2.0 ** -24 * size
    bound += R.HALF_STEP[F16] * (np.abs(whole) + bound) + R.TINY[F16]
    assert np.all(np.abs(grad - whole) <= bound), float(np.max(np.abs(grad - whole) / bound))
    # the step on that gradient, bit for bit
    g16 = t.dev.to_host(t.d_g, vocab * dim, np.uint16)
    w, m, v = t.master.reshape(-1).copy(), np.zeros(vocab * dim, np.float32), np.zeros(vocab * dim, np.float32)
    p16 = oracle.f32_to_f16(w)
    st = oracle.new_loss_scale()
    oracle.mixed_adam_step([g16], [w], [m], [v], [p16], 1e-3, 0.9, 0.999, 1e-8, 0.0, st)
    assert np.array_equal(t.dev.to_host(t.d_w, vocab * dim).view(np.uint32), w.view(np.uint32))
    assert np.array_equal(t.dev.to_host(t.d_p, vocab * dim, np.uint16), p16)
    assert t.state().adam_t == st.adam_t == 1
    t.close()


@pytest.mark.gpu
def test_an_overflowing_gradient_is_skipped_and_the_next_one_fits(gm, dev):
    """With a loss scale that no fp16 gradient survives, the step is skipped on the device and the scale falls."""
    t = Tied(gm, dev, 64, 32, 50, scale0=2.0 ** 24)
    before = t.dev.to_host(t.d_w, 50 * 32)
    t.step()
    assert not np.isfinite(t.get(t.d_g, (50, 32))).all()
    st = t.state()
    assert st.last_overflow == 1 and st.skipped == 1 and st.adam_t == 0 and st.scale == 2.0 ** 23
    assert np.array_equal(t.dev.to_host(t.d_w, 50 * 32), before)
    for _ in range(20):
        t.step()
    st = t.state()
    assert st.last_overflow == 0 and st.adam_t > 0 and np.isfinite(t.dev.to_host(t.d_w, 50 * 32)).all()
    assert gm.lib.gm_linear_xent_status(dev.h) == 0
    t.close()


@pytest.mark.gpu
def test_one_graph_of_the_whole_step(gm, dev):
    """Captured once and replayed: the same parameters as the same number of eager steps."""
    a, b = Tied(gm, dev, 150, 48, 400), Tied(gm, dev, 150, 48, 400)
    for _ in range(4):
        a.step()
    b.step()                                       # warm: kernels loaded, lists built
    dev.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(gm.lib.gm_device_stream(dev.h))):
        b.step()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for x, y in ((a.d_w, b.d_w), (a.d_m, b.d_m), (a.d_v, b.d_v)):
        assert np.array_equal(dev.to_host(x, 400 * 48), dev.to_host(y, 400 * 48))
    assert a.state().adam_t == b.state().adam_t == 4
    del g
    a.close()
    b.close()
