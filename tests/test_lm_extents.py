"""Matrices whose last byte lies beyond what 64 bits count are refused, not taken for small ones."""
import pytest

MOST = (1 << 31) - 1


def embedding(gm, dtype, tokens, vocab, ld_table, ld_out):
    return gm.Embedding(dtype=dtype, tokens=tokens, dim=16, vocab=vocab, ld_table=ld_table, ld_out=ld_out, padding_token=-1, scale=1.0)


@pytest.mark.parametrize("dtype", [0, 2, 4])
def test_sizes_that_overflow_need_no_device(gm, dtype):
    size = gm.lib.gm_embedding_workspace_bytes
    assert size(embedding(gm, dtype, 4, 8, MOST, 16)) > 0                 # a wide stride alone is none
    assert size(embedding(gm, dtype, 4, 1 << 28, MOST, 16)) > 0           # 2^59 elements
    for e in (embedding(gm, dtype, 4, MOST - 1, MOST, 16), embedding(gm, dtype, MOST, 8, 16, MOST), embedding(gm, dtype, 4, 1 << 30, MOST, 16)):
        assert size(e) == -1 and "elements" in gm.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [0, 2, 4])
def test_calls_refuse_them(gm, dev, dtype):
    L = gm.lib
    a, b, tok, ws = (dev.alloc(k) for k in (1 << 12, 1 << 12, 64, 1 << 16))
    before = L.gm_device_launch_count(dev.h)
    assert L.gm_dropout_async(dev.h, dtype, MOST, 16, a, MOST, 0, 0, b, MOST, gm.dropout(0.5, 1)) == -9
    assert L.gm_dropout_async(dev.h, dtype, MOST, 16, a, MOST, b, MOST, a, MOST, gm.dropout(0.5, 1)) == -9
    e = embedding(gm, dtype, 4, MOST - 1, MOST, 16)
    assert L.gm_embedding_forward_async(dev.h, e, a, tok, b, None) == -9
    assert L.gm_embedding_backward_async(dev.h, e, tok, b, None, a, dtype, 1, ws, 1 << 16) == -9
    assert L.gm_device_launch_count(dev.h) == before
    for p in (a, b, tok, ws):
        dev.free(p)
