"""The language-model operators where element offsets pass 32 bits, and from two device handles at once."""
import numpy as np
import pytest
import torch

import lm_ref as R

BF16 = 4


def P(t):
    return t.data_ptr()


@pytest.mark.gpu
def test_dropout_with_rows_gigabytes_apart(gm, dev):
    rows, cols, ld = 3, 72, 1_500_000_000                      # the last row begins 3e9 elements in
    x = torch.empty(2 * ld + cols, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    v = torch.as_strided(x, (rows, cols), (ld, 1))
    v.normal_()
    torch.cuda.synchronize()
    gm.check(gm.lib.gm_dropout_async(dev.h, BF16, rows, cols, P(x), ld, 0, cols, P(y), cols, gm.dropout(0.5, 3, 4)))
    dev.sync()
    keep, up = R.keep_mask(rows * cols, 0.5, 3, 4)
    want = np.where(keep.reshape(rows, cols), v.float().cpu().numpy() * up, np.float32(0))
    assert np.array_equal(y.double().cpu().numpy(), R.rounded(want, BF16))


@pytest.mark.gpu
def test_embedding_of_a_table_beyond_32_bits(gm, dev):
    vocab, dim, n = 600_000, 4096, 50                           # 2.46e9 elements
    L = gm.lib
    table = torch.empty(vocab, dim, dtype=torch.bfloat16, device="cuda").normal_()
    tok = torch.cat([torch.tensor([vocab - 1, 0, vocab - 1, 524_288, 524_287]), torch.randint(0, vocab, (n - 5,))]).int().cuda()
    out, dout = torch.empty(n, dim, dtype=torch.bfloat16, device="cuda"), torch.empty(n, dim, dtype=torch.bfloat16, device="cuda").normal_()
    grad = torch.full((vocab, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    e = gm.Embedding(dtype=BF16, tokens=n, dim=dim, vocab=vocab, ld_table=dim, ld_out=dim, padding_token=-1, scale=1.0)
    room = torch.empty(L.gm_embedding_workspace_bytes(e), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    gm.check(L.gm_embedding_forward_async(dev.h, e, P(table), P(tok), P(out), None))
    gm.check(L.gm_embedding_backward_async(dev.h, e, P(tok), P(dout), None, P(grad), BF16, 0, P(room), room.numel()))
    dev.sync()
    t = tok.long()
    assert torch.equal(out, table[t])
    want = torch.zeros(vocab, 1, dtype=torch.bool, device="cuda")
    want[t] = True
    assert torch.equal((grad != 0).any(1, keepdim=True), want)
    pair = dout[t == vocab - 1].float().sum(0)                  # two or more rows; a sum of L is L - 1 roundings in binary32, one to bf16
    assert torch.all((grad[vocab - 1].float() - pair).abs() <= 2.0 ** -8 * pair.abs() + n * 2.0 ** -23 * dout.float().abs().sum(0))
    single = torch.tensor([k for k in range(n) if int((t == t[k]).sum()) == 1], device="cuda")
    assert torch.equal(grad[t[single]], dout[single])


@pytest.mark.gpu
def test_loss_over_a_table_beyond_32_bits(gm, dev):
    """Losses of every row, and the gradient of the table's last rows, against 64 bits."""
    vocab, dim, n = 540_000, 4096, 140                          # 2.2e9 elements
    L = gm.lib
    w = torch.empty(vocab, dim, dtype=torch.bfloat16, device="cuda").normal_(0, dim ** -0.5)
    x = torch.empty(n, dim, dtype=torch.bfloat16, device="cuda").normal_()
    t = torch.randint(0, vocab, (n,), device="cuda", dtype=torch.int32)
    t[:4] = torch.tensor([vocab - 1, 524_288, 524_287, 0])
    h = gm.LinearXent(dtype=BF16, tokens=n, dim=dim, vocab=vocab, ld_hidden=dim, ld_weight=dim, mean=0)
    room = torch.empty(L.gm_linear_xent_workspace_bytes(h, 1), dtype=torch.uint8, device="cuda")
    losses, lse, total = (torch.empty(k, device="cuda") for k in (n, n, 2))
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    torch.cuda.synchronize()
    gm.check(L.gm_linear_xent_forward_async(dev.h, h, P(x), P(w), P(t), P(losses), P(lse), P(total), P(room), room.numel()))
    gm.check(L.gm_linear_xent_backward_async(dev.h, h, P(x), P(w), P(t), P(lse), 0, 1.0, P(dx), P(dw), 0, P(room), room.numel()))
    dev.sync()
    assert L.gm_linear_xent_status(dev.h) == 0
    X, parts = x.double(), []
    for a in range(0, vocab, 60_000):
        parts.append(torch.logsumexp(X @ w[a:a + 60_000].double().T, 1))
    want = torch.logsumexp(torch.stack(parts), 0)
    z = (X * w[t.long()].double()).sum(1)
    size = (X.abs() * w[t.long()].double().abs()).sum(1).max()
    bound = 2 * ((dim + 8) * 2.0 ** -23 * size + 2.0 ** -22 * (want.abs().max() + 16) + (256 + vocab / 2048) * 2.0 ** -24)
    assert torch.all((lse.double() - want).abs() <= bound) and torch.all((losses.double() - (want - z)).abs() <= bound)
    for a, b in ((vocab - 300, vocab), (524_200, 524_400), (0, 100)):
        s = torch.exp(X @ w[a:b].double().T - want[:, None])
        for k in range(n):
            if a <= int(t[k]) < b:
                s[k, int(t[k]) - a] -= 1
        ref, mag = s.T @ X, s.abs().T @ X.abs()
        # probabilities off by `bound`, S rounded once, sums of n terms, one rounding
        err = (dw[a:b].double() - ref).abs()
        assert torch.all(err <= (2.0 ** -8 + bound + (n + 16) * 2.0 ** -23) * 1.01 * mag + 2.0 ** -8 * (ref.abs() + mag * 2.0 ** -7)), float(err.max())


@pytest.mark.gpu
def test_two_device_handles_at_once(gm, dev):
    """Two handles have two streams: the same calls in flight together, each with its own workspace, give
    what they give alone."""
    L = gm.lib
    other = gm.Device(L.gm_device_ordinal(dev.h))
    n, dim, vocab = 700, 136, 5000
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(n, dim, generator=g, device="cuda").half()
    w = (torch.randn(vocab, dim, generator=g, device="cuda") / 12).half()
    t = torch.randint(-50, vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    h = gm.LinearXent(dtype=2, tokens=n, dim=dim, vocab=vocab, ld_hidden=dim, ld_weight=dim, mean=1)
    e = gm.Embedding(dtype=2, tokens=n, dim=dim, vocab=vocab, ld_table=dim, ld_out=dim, padding_token=-1, scale=1.0)

    def make():
        s = [torch.empty(k, device="cuda") for k in (n, n, 2)]
        return s + [torch.empty_like(x), torch.empty_like(w), torch.empty_like(w),
                    torch.empty(max(L.gm_linear_xent_workspace_bytes(h, 2), L.gm_embedding_workspace_bytes(e), L.gm_linear_xent_workspace_bytes(h, 0)),
                                dtype=torch.uint8, device="cuda")]

    def go(d, b):
        losses, lse, total, dx, dw, de, room = b
        gm.check(L.gm_linear_xent_forward_async(d.h, h, P(x), P(w), P(t), P(losses), P(lse), P(total), P(room), room.numel()))
        gm.check(L.gm_linear_xent_backward_async(d.h, h, P(x), P(w), P(t), P(lse), 0, 64.0, P(dx), P(dw), 0, P(room), room.numel()))
        gm.check(L.gm_embedding_backward_async(d.h, e, P(t), P(dx), gm.dropout(0.2, 1), P(de), 2, 0, P(room), room.numel()))
    alone, a, b = make(), make(), make()
    torch.cuda.synchronize()
    go(dev, alone)
    torch.cuda.synchronize()
    for _ in range(20):
        go(dev, a)
        go(other, b)
    torch.cuda.synchronize()
    for p, q, r in zip(alone[:-1], a, b):
        assert torch.equal(p, q) and torch.equal(p, r)
    assert L.gm_linear_xent_status(other.h) == 0
    other.close()
