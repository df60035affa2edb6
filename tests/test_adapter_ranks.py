"""Ranks of very different sizes in one LoRA branch: each rank's gradients keep their own precision.

The bounds are those of tests/test_adapter.py: 2^-19 of the sum of the magnitudes of an entry's own
terms (dA[j, c] and dB[o, j] hold terms of rank j only)."""

import pytest
import torch

from test_adapter import _branch_inputs, _check_branch, _run_branch


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [2, 16, 40])
@pytest.mark.parametrize("power", [-24, -36, -60, 40])
def test_ranks_far_from_one_another(power, rank):
    """Every second column of B, then every second row of A, scaled: as a decayed or pruned rank beside a
    live one."""
    x, base, a, b, g = _branch_inputs(300, 136, 264, rank, 40 + rank)
    for scale_a, scale_b in ((False, True), (True, False), (True, True)):
        a2, b2 = a.clone(), b.clone()
        if scale_a:
            a2[::2] *= 2.0 ** power
        if scale_b:
            b2[:, 1::2] *= 2.0 ** power
        out = _run_branch(x, base, a2, b2, 2.0, 0.1, 6, g)
        keep = (out[0].float().isfinite().all() and out[1].float().isfinite().all())
        if keep:  # y and dx pass fp16's range where a rank is scaled up
            _check_branch(x, base, a2, b2, 2.0, 0.1, 6, g, *out)
        else:
            _check_branch(x, base, a2, b2, 2.0, 0.1, 6, g, *_exact_fp16(x, base, a2, b2, g), *out[2:])


def _exact_fp16(x, base, a, b, g):
    """Stand-ins for y and dx that have passed fp16's range: the exact values (only dA and dB are
    checked then)."""
    from oracle import adapter as oracle

    host = [t.detach().double().cpu().numpy() for t in (x, base, a, b, g)]
    want, _ = oracle.branch(*host[:4], 2.0, 0.1, 6, host[4])
    return torch.from_numpy(want[0]), torch.from_numpy(want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_an_infinite_rank_leaves_the_others(p):
    """An infinity in one row of A makes that rank's t, and with it dB's column, infinite or NaN, one in
    a column of B its dt and dA's row; the other ranks' gradients keep their bits, small as they are."""
    x, base, a, b, g = _branch_inputs(300, 136, 264, 8, 9)
    a, b = a * 2.0 ** -20, b * 2.0 ** -20
    want = _run_branch(x, base, a, b, 1.0, p, 6, g)
    others = [j for j in range(8) if j != 3]
    a2, b2 = a.clone(), b.clone()
    a2[3, 7], b2[11, 3] = float("inf"), float("inf")
    got = _run_branch(x, base, a2, b, 1.0, p, 6, g)
    assert torch.equal(got[3][:, others], want[3][:, others])
    assert not torch.isfinite(got[3][:, 3]).any()
    assert torch.equal(got[2], want[2])          # dA does not depend on A
    got = _run_branch(x, base, a, b2, 1.0, p, 6, g)
    assert torch.equal(got[2][others], want[2][others])
    assert not torch.isfinite(got[2][3]).any()
    assert torch.equal(got[3], want[3])
