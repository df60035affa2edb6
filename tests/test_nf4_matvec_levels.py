"""The levels of the few-row NF4 product: as exact as the fp32 values that a group holds, whatever the
table, and the same in both of its kernels.

Error bound, from the arithmetic: one rounding to fp16 (2^-11 of the result, 2^-25 below the normal
range); the levels in two fp16 parts keep 2^-22 of each term, and fp32 products and sums add 2^-20
of the sum of the terms' magnitudes, 2^-19 in all. (A level of one fp16 number is off by up to 2^-11
of its terms: with 64 to 320 terms an output that happens to be small shows 2^-14 of them.)"""

import numpy as np
import pytest
import torch

from talm_b200 import nf4_dequant, qgroup

NF4 = qgroup.NF4_LEVELS
TABLES = {
    "nf4": NF4,
    "powers": [(-1.0) ** i * 2.0 ** -i for i in range(16)],
    "large": [1.0e5 * v for v in NF4],                   # beyond fp16's range
    "huge": [2.0e30 * v for v in NF4],
    "tiny": [3.0e-30 * v for v in NF4],
    "uneven": [0.0, 1e-6, -1e-6, 3e-5, -7e-4, 0.01, 0.1, 1 / 3, 1.7, -2.3, 9.1, 33.3, -100.1, 900.7,
               -3000.3, 0.7],
    "one": [0.1] * 16,
    "zero": [0.0] * 16,
}


def _case(rows, n_out, n_in, levels, seed, codes=None, x=None, scale=None):
    """Arrays of a grouped weight with that table, and the float64 product with its bound."""
    g = torch.Generator().manual_seed(seed)
    n = n_out * n_in
    blocks = n // 64
    x = torch.randn(rows, n_in, generator=g).half() if x is None else x
    choices = torch.arange(16) if codes is None else torch.tensor(codes)
    code = choices[torch.randint(0, len(choices), (n,), generator=g)]
    packed = (code[0::2] * 16 + code[1::2]).to(torch.uint8)
    absmax8 = torch.randint(0, 256, (blocks,), generator=g, dtype=torch.uint8)
    table8 = torch.sort(torch.rand(256, generator=g) * 2 - 1).values
    n2 = -(-blocks // 256)
    absmax2, offset2 = torch.rand(n2, generator=g) * 0.01, torch.rand(n2, generator=g) * 0.03 + 0.01
    if scale is not None:  # keeps the result in fp16's range where the table is far from one
        absmax2, offset2 = absmax2 * scale, offset2 * scale
    second = torch.arange(blocks) // 256
    s = (table8[absmax8.long()] * absmax2[second] + offset2[second]).double()
    levels = torch.tensor(levels, dtype=torch.float32)
    w = (levels.double()[code] * s.repeat_interleave(64)).view(n_out, n_in)
    y = x.double() @ w.t()
    total = x.double().abs() @ w.abs().t()
    tol = 2.0 ** -11 * y.abs() + 2.0 ** -25 + 2.0 ** -19 * total
    arrays = [t.cuda() for t in (packed, absmax8, table8, absmax2, offset2, levels)]
    return x.cuda(), arrays, y, tol


def _run(x, arrays, n_out, n_in):
    out = torch.empty(x.shape[0], n_out, dtype=torch.float16, device="cuda")
    packed, absmax8, table8, absmax2, offset2, levels = arrays
    return qgroup.launch_matvec(x, packed, absmax8, table8, absmax2, offset2, levels, out, 0, n_out,
                                n_in, 64, 256)


def _off(got, y, tol):
    return float(((got.double().cpu() - y).abs() / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [None, (6, 7, 8), (1, 14), (7, 8)], ids=str)
@pytest.mark.parametrize("n_in", [64, 192, 320])
@pytest.mark.parametrize("rows", [1, 2, 9, 17, 32])
def test_levels_are_kept_as_the_table_gives_them(rows, n_in, codes):
    """Many outputs, small ones among them; codes of all levels, and of the smallest ones only."""
    x, arrays, y, tol = _case(rows, 2053, n_in, NF4, rows + n_in, codes)
    assert _off(_run(x, arrays, 2053, n_in), y, tol) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 9, 32])
@pytest.mark.parametrize("table", TABLES)
def test_any_table(table, rows):
    """Sixteen levels of any size: beyond fp16's range, far below it, of very different sizes."""
    levels = TABLES[table]
    most = max(abs(v) for v in levels)
    scale = None if not most or 1e-3 < most < 1e4 else float(np.float32(1 / most))
    x, arrays, y, tol = _case(rows, 200, 192, levels, rows, scale=scale)
    assert _off(_run(x, arrays, 200, 192), y, tol) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 13, 32])
def test_both_kernels_give_the_same_product(rows):
    """Packed bytes off their 16-byte boundary go to the byte-wise kernel: the two differ by fp32
    summation order only, so hardly a rounding falls the other way."""
    x, arrays, y, tol = _case(rows, 1500, 320, NF4, 5)
    wide = _run(x, arrays, 1500, 320)
    moved = torch.empty(arrays[0].numel() + 1, dtype=torch.uint8, device="cuda")[1:]
    narrow = _run(x, [moved.copy_(arrays[0]), *arrays[1:]], 1500, 320)
    assert _off(narrow, y, tol) <= 1
    # a value is rounded the other way when a border lies within the two errors (2^-19 of its terms,
    # some 2^-15 of the value at 320 terms) of it: under one in 16
    assert float((wide != narrow).float().mean()) < 1 / 16


@pytest.mark.gpu
def test_rounded_like_the_exact_product():
    """1536 terms: nearly every output is the exact product's nearest fp16 number. (The share that is
    not is twice the error over the step: 2^-19 of the terms' norm at most, a step of 2^-11: 2^-7
    with norm for value, four times that with small values. Levels of one fp16 number gave 1 in 8.)"""
    x, arrays, y, _ = _case(4, 4096, 1536, NF4, 8)
    got = _run(x, arrays, 4096, 1536).cpu()
    assert float((got != y.half()).float().mean()) < 4 * 2.0 ** -7


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 9])
def test_infinite_inputs_meet_every_level(rows):
    """An infinity times a level is an infinity of the product's sign, whatever parts the level is
    held in; times the level zero it is NaN."""
    for code, level in enumerate(NF4):
        packed = torch.full((8 * 32,), code * 17, dtype=torch.uint8, device="cuda")
        absmax = torch.full((8,), 0.5, device="cuda")
        for sign in (1, -1):
            x = torch.zeros(rows, 64, dtype=torch.float16, device="cuda")
            x[0, 5] = sign * float("inf")
            y = nf4_dequant.nf4_matvec(x, packed, absmax, 64)
            if level == 0:
                assert torch.isnan(y[0]).all()
            else:
                assert (y[0] == sign * np.sign(level) * float("inf")).all(), code
            assert not y[1:].any()
