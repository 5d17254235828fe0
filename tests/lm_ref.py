"""Plain host restatements of the language-model operators, in 64 bits, and the
conversions between numpy arrays and the element types of the library."""
import numpy as np
import torch

TORCH = {0: torch.float32, 2: torch.float16, 4: torch.bfloat16}
HALF_STEP = {0: 2.0 ** -24, 2: 2.0 ** -11, 4: 2.0 ** -8}       # relative rounding error of a store
TINY = {0: 2.0 ** -150, 2: 2.0 ** -25, 4: 2.0 ** -134}         # half the spacing of the subnormals


def bytes_of(x, dtype):
    """The array's values in the element type, as raw bytes for an upload."""
    return torch.from_numpy(np.ascontiguousarray(x)).to(TORCH[dtype]).contiguous().view(torch.uint8).numpy().reshape(-1)


def rounded(x, dtype):
    """The values the element type can hold, as float64."""
    return torch.from_numpy(np.ascontiguousarray(x)).to(TORCH[dtype]).double().numpy()


def values_of(raw, dtype):
    """float64 values of raw bytes."""
    return torch.from_numpy(np.ascontiguousarray(raw)).view(TORCH[dtype]).double().numpy()


def eb(dtype):
    return 4 if dtype == 0 else 2


def philox(c0, c1, c2, c3, k0, k1, rounds=10):
    """Philox-4x32 on arrays of uint64 that hold 32-bit words."""
    low, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.asarray(x, np.uint64) for x in (c0, c1, c2, c3)]
    for _ in range(rounds):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> sh) ^ c[1] ^ np.uint64(k0), b & low, (a >> sh) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def keep_mask(n, p, seed, offset):
    """Which of n elements stay, and the factor of those (a binary32 number)."""
    cut = int(np.floor(float(np.float32(p)) * 65536.0 + 0.5))
    offset &= (1 << 64) - 1
    block = np.arange((n + 7) // 8, dtype=np.uint64)
    o = np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)
    w = philox(block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), o[0], o[1], seed & 0xFFFFFFFF, seed >> 32)
    lanes = np.stack([x for c in w for x in (c & np.uint64(0xFFFF), c >> np.uint64(16))], axis=1).reshape(-1)[:n]
    return lanes >= cut, np.float32(65536.0 / (65536 - cut)) if cut < 65536 else np.float32(0.0)


def strided(x, ld, dtype, fill=-7.0):
    """A matrix with its rows `ld` apart, as the flat values a buffer holds."""
    out = np.full((x.shape[0], ld), fill, np.float64)
    out[:, :x.shape[1]] = x
    return out.reshape(-1)
