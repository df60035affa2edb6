"""CPU oracle of the adapted 4-bit projection: Philox masks (integers, exact), the LoRA branch with
its gradients and the few-row NF4 product, in float64 from their definitions.

`philox4x32` is the generator of Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
1, 2, 3" (2011), with a given number of rounds.
"""

import numpy as np

from . import nf4

DROP_ALL = 32768


def philox4x32(counter, key, rounds):
    """counter: four arrays of uint32, key: two ints -> the four result words (uint32 arrays)."""
    mask = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(rounds):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & mask,
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & mask]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return [v.astype(np.uint32) for v in c]


def keep_mask(n, p, seed, first=0):
    """Which of the elements first .. first + n - 1 (first a multiple of 8) are kept, and the
    factor that scales them."""
    q = np.arange(first // 8, first // 8 + -(-n // 8), dtype=np.uint64)
    zero = np.zeros_like(q)
    words = philox4x32((q & np.uint64(0xFFFFFFFF), q >> np.uint64(32), zero, zero),
                       (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF), 7)
    halves = np.stack([h for w in words for h in (w & np.uint32(0x7FFF),
                                                  (w >> np.uint32(16)) & np.uint32(0x7FFF))], 1)
    drop = int(np.floor(p * DROP_ALL + 0.5))
    return halves.reshape(-1)[:n] >= drop, DROP_ALL / (DROP_ALL - drop) if drop < DROP_ALL else 0.0


def branch(x, base, a, b, scaling, p, seed, g):
    """The branch in float64 on arrays (x [T, in], base and g [T, out], a [r, in], b [out, r]):
    y, dx, da, db and the sums of magnitudes that bound a kernel's rounding errors
    (of y's branch, dx, da and db)."""
    x, base, a, b, g = (np.asarray(v, dtype=np.float64) for v in (x, base, a, b, g))
    if p > 0:
        kept, factor = keep_mask(x.size, p, seed)
        m = kept.reshape(x.shape) * factor
    else:
        m = np.ones_like(x)
    xd = np.where(m > 0, x, 0.0) * m
    t, dt = xd @ a.T, scaling * (g @ b)
    out = (base + scaling * (t @ b.T), (dt @ a) * m, dt.T @ xd, scaling * (g.T @ t))
    at, adt = np.abs(xd) @ np.abs(a).T, abs(scaling) * (np.abs(g) @ np.abs(b))
    sums = (abs(scaling) * (at @ np.abs(b).T), (adt @ np.abs(a)) * m, adt.T @ np.abs(xd),
            abs(scaling) * (np.abs(g).T @ at))
    return out, sums


def nf4_weight(packed, scales, n_out, n_in, blocksize):
    """The float64 weight [n_out, n_in]: level times the fp32 scale of the element's block of the
    flattened weight, not rounded."""
    n = n_out * n_in
    scale = np.asarray(scales, dtype=np.float32).astype(np.float64)[np.arange(n) // blocksize]
    return (nf4.unpack_levels(packed, n).astype(np.float64) * scale).reshape(n_out, n_in)


def double_quant_scales(absmax8, code, absmax2, offset2, row0, qblock2):
    """fp32(fp32(code[absmax8] * absmax2) + offset2), the second level at (row0 + i) / qblock2."""
    second = (np.arange(len(absmax8)) + row0) // qblock2
    product = (np.asarray(code, np.float32)[absmax8] * np.asarray(absmax2, np.float32)[second])
    return (product + np.asarray(offset2, np.float32)[second]).astype(np.float32)
