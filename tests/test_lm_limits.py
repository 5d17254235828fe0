"""Sizes of the vocabulary loss beyond which it refuses, told without a device."""


def test_rows_whose_gradient_would_outlast_the_bounded_waits(gm):
    size = gm.lib.gm_linear_xent_workspace_bytes

    def loss(tokens, vocab=1000, dim=8):
        return gm.LinearXent(dtype=2, tokens=tokens, dim=dim, vocab=vocab, ld_hidden=dim, ld_weight=dim, mean=1)
    for which in (0, 1, 2):
        assert size(loss(1 << 26), which) > 0
        assert size(loss((1 << 26) + 1), which) == -1 and "too many" in gm.last_error()
        assert size(loss(100, 1 << 28), which) > 0
        assert size(loss(100, (1 << 28) + 1), which) == -1
        assert size(loss(100, 1000, 1 << 24), which) > 0
        assert size(loss(100, 1000, (1 << 24) + 8), which) == -1
