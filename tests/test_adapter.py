"""Counter-based dropout and the LoRA branch against a float64 oracle.

Error bounds, from the arithmetic. Dropout: one fp32 product of an exact mask, rounded once: half a
step of the type, plus 2^-24 for the fp32 factor and 2^-24 for the product. Branch: y and dx are
rounded to fp16 once (2^-11 of the value, 2^-25 below the normal range); their rank-wide products
run on operands split in two bf16 parts with the product of the two small parts left out, 2^-16 of
the sum of the terms' magnitudes (3 * 2^-18 for the parts' own rounding and the product left out).
t, dt, dA and dB run on fp16 activations as they are and fp32 operands split in two fp16 parts
(2^-22 of each), with fp32 sums in short runs: 2^-19 of the sum of magnitudes."""

import math

import numpy as np
import pytest
import torch

from oracle import adapter as oracle
from talm_b200 import _lib, adapter, build, nf4_format, qgroup, qlora

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


# ------------------------------------------------------------------------------------------
# on the CPU: the generator, the refusals
# ------------------------------------------------------------------------------------------
def test_oracle_generator_gives_the_published_vectors():
    """Philox4x32 known answers (counter and key of zeros, 7 and 10 rounds)."""
    zero = [np.zeros(1, np.uint64)] * 4
    words = [int(w[0]) for w in oracle.philox4x32(zero, (0, 0), 7)]
    assert words == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    words = [int(w[0]) for w in oracle.philox4x32(zero, (0, 0), 10)]
    assert words == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


def test_oracle_mask_has_the_asked_share_and_no_pattern():
    """Shares within five standard deviations, for elements of every place in their group of eight
    and for neighbours together (which are independent)."""
    n, p = 1 << 20, 0.25
    kept, factor = oracle.keep_mask(n, p, 0x1234567890ABCDEF)
    assert factor == 4 / 3
    sigma = math.sqrt(p * (1 - p) / (n / 8))
    shares = kept.reshape(-1, 8).mean(0)
    assert (np.abs(shares - 0.75) < 5 * sigma).all()
    both = (kept[1:] & kept[:-1]).mean()
    assert abs(both - 0.75 ** 2) < 5 * math.sqrt(0.5625 * 0.4375 / n) * 2
    assert not np.array_equal(kept, oracle.keep_mask(n, p, 0x1234567890ABCDEE)[0])
    tail = oracle.keep_mask(64, p, 5, first=1 << 20)[0]
    assert np.array_equal(tail, oracle.keep_mask((1 << 20) + 64, p, 5)[0][1 << 20:])


def test_thresholds():
    assert [adapter.drop_threshold(p) for p in (0, 1, 0.5, 0.05, 1e-9)] == [0, 32768, 16384, 1638, 0]
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="between 0 and 1"):
            adapter.drop_threshold(p)


def test_c_entries_reject_bad_arguments(lib):
    def drop(n_rows=1, n_cols=8, ld=8, dtype=0, drop=5, seed=16):
        return lib.talm_dropout(None, ld, n_rows, n_cols, dtype, seed, drop, None, None)
    assert drop(drop=-1) == 1 and drop(drop=32769) == 1 and drop(seed=None) == 1
    assert drop(n_rows=-1) == 1 and drop(ld=7) == 1 and drop(dtype=3) == 1
    assert drop() == 1 and b"null" in lib.talm_last_error()
    assert drop(n_rows=0) == 0 and drop(n_cols=0, ld=0) == 0
    assert drop(n_rows=1 << 40, n_cols=1 << 20, ld=1 << 20) == 3

    size = _lib._SZ(0)
    assert lib.talm_lora_sizes(4, 64, 64, 16, size, size, size) == 0
    for bad in ((-1, 64, 64, 16), (4, 60, 64, 16), (4, 64, 60, 16), (4, 64, 64, 0),
                (4, 64, 64, 65), (4, 0, 64, 16)):
        assert lib.talm_lora_sizes(*bad, size, size, size) == 1, bad
    assert lib.talm_lora_sizes(1 << 31, 64, 64, 16, size, size, size) == 3

    def forward(n_rows=4, drop=0, seed=None, ptr=None, ld_x=64, saved=1 << 20, ws=1 << 24):
        return lib.talm_lora_forward(ptr, ld_x, ptr, 64, ptr, ptr, n_rows, 64, 64, 16, 1.0, seed,
                                     drop, ptr, ptr, saved, ptr, ws, None)
    assert forward() == 1 and forward(drop=5) == 1 and forward(n_rows=0) == 0
    assert forward(ptr=8) == 1                      # rows off their 16-byte boundary
    assert forward(ptr=16, ld_x=60) == 1 and forward(ptr=16, ld_x=68) == 1
    assert forward(ptr=16, saved=3) == 1 and b"too small" in lib.talm_last_error()
    assert forward(ptr=16, ws=3) == 1

    def backward(n_rows=4, ptr=None, out=16, ws=1 << 24, ld_g=64):
        return lib.talm_lora_backward(ptr, ld_g, ptr, 64, ptr, 1 << 24, n_rows, 64, 64, 16,
                                       1.0, None, 0, out, None, None, ptr, ws, None)
    assert backward() == 1
    assert backward(out=None) == 0                  # nothing asked for
    assert backward(ptr=16, ld_g=60) == 1 and backward(ptr=16, ws=3) == 1


def test_python_entries_refuse_what_the_kernels_do_not_take():
    x, base = torch.zeros(4, 64).half(), torch.zeros(4, 32).half()
    a, b = torch.zeros(8, 64), torch.zeros(32, 8)
    seed = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(TypeError):
        adapter.dropout(x.double(), 0.1, seed)
    with pytest.raises(RuntimeError, match="CUDA"):
        adapter.dropout(x, 0.1, seed)
    with pytest.raises(RuntimeError, match="CUDA"):
        adapter.lora_branch(x, base, a, b, 1.0)
    with pytest.raises(TypeError):
        adapter.lora_branch(x.float(), base, a, b, 1.0)
    with pytest.raises(TypeError):
        adapter.lora_branch(x, base, a.half(), b, 1.0)
    with pytest.raises(ValueError, match="rows"):
        adapter.lora_branch(x[:3], base, a, b, 1.0)
    with pytest.raises(ValueError, match="map"):
        adapter.lora_branch(x, base, a, b[:, :4], 1.0)
    with pytest.raises(ValueError, match="multiples"):
        adapter.lora_branch(x[:, :60], base, a[:, :60], b, 1.0)
    with pytest.raises(ValueError, match="rank"):
        adapter.lora_branch(x, base, torch.zeros(65, 64), torch.zeros(32, 65), 1.0)
    with pytest.raises(ValueError, match="between"):
        adapter.lora_branch(x, base, a, b, 1.0, p=1.5)


def test_fused_adapters_are_opt_in():
    config = qlora.qwen25_15b_config(vocab_size=64, hidden_size=512, intermediate_size=1024,
                                     num_hidden_layers=1, num_attention_heads=8,
                                     num_key_value_heads=2)
    for fused in (False, True):
        model = qlora.build_model(config, "cpu", lora_fused=fused) if fused \
            else qlora.build_model(config, "cpu")
        found = [m for m in model.modules() if isinstance(m, qlora.LoraLinear)]
        assert len(found) == 2 and all(m.fused is fused for m in found)


# ------------------------------------------------------------------------------------------
# dropout
# ------------------------------------------------------------------------------------------
def _seed(value):
    return torch.tensor([value], dtype=torch.int64, device="cuda")


def _check_dropout(x, y, p, seed):
    kept, factor = oracle.keep_mask(x.numel(), p, seed)
    xs = x.detach().double().cpu().numpy().reshape(-1)
    got = y.detach().double().cpu().numpy().reshape(-1)
    want = np.where(kept, xs, 0.0) * factor
    half = HALF_STEP[x.dtype]
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
    assert y.dtype == x.dtype and y.shape == x.shape
    assert not got[~kept].any() and not np.signbit(got[~kept]).any()
    assert (np.abs(got - want) <= (half + 2 * 2.0 ** -24) * np.abs(want) + tiny[x.dtype]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(HALF_STEP), ids=str)
@pytest.mark.parametrize("shape", [(), (1,), (7,), (8,), (9,), (3, 5), (1, 1537), (37, 64),
                                   (5, 3, 72), (129, 255), (1126, 1536)], ids=str)
def test_dropout_matches_the_oracle(shape, dtype):
    g = torch.Generator("cuda").manual_seed(len(shape))
    for p, seed in ((0.05, 3), (0.5, (1 << 62) + 12345), (0.0, 1), (0.999, 7)):
        x = torch.randn(shape, generator=g, device="cuda").to(dtype)
        _check_dropout(x, adapter.dropout(x, p, _seed(seed)), p, seed)
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_dropout_of_everything_and_of_nothing():
    x = torch.randn(65, 33, device="cuda")
    x[0, 0], x[1, 1], x[2, 2] = float("nan"), float("inf"), -float("inf")
    y = adapter.dropout(x, 1.0, _seed(4))
    assert not y.any() and not torch.signbit(y).any()      # whatever it held, also infinities
    y = adapter.dropout(x, 0.0, _seed(4))
    assert torch.equal(y[3:], x[3:]) and torch.isnan(y[0, 0]) and torch.isinf(y[1, 1])
    assert adapter.dropout(x[:0], 0.5, _seed(4)).shape == (0, 33)
    assert adapter.dropout(x[:, :0], 0.5, _seed(4)).shape == (65, 0)
    with pytest.raises(ValueError, match="seed"):
        adapter.dropout(x, 0.5, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="seed"):
        adapter.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(HALF_STEP), ids=str)
def test_dropout_strides_and_gradients(dtype):
    """The mask goes by the element's index, not by where it lies: rows of a wider tensor, a
    transposed and a broadcast one; the gradient is the same map, also of broadcast gradients, and
    once more."""
    wide = torch.randn(40, 90, device="cuda").to(dtype)
    for x in (wide[:, 3:80], wide[:, 8:72], wide.t(), wide[:1].expand(40, 90), wide[::3, ::2],
              wide.view(5, 8, 90).transpose(0, 1)):
        _check_dropout(x, adapter.dropout(x, 0.3, _seed(9)), 0.3, 9)
    x = wide.clone().requires_grad_()
    y = adapter.dropout(x, 0.3, _seed(9))
    g = torch.randn_like(x)
    dx, = torch.autograd.grad(y, x, g, retain_graph=True)
    _check_dropout(g, dx, 0.3, 9)
    dx, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    _check_dropout(torch.ones_like(x), dx, 0.3, 9)
    v = torch.randn_like(x).requires_grad_()
    dx, = torch.autograd.grad(y, x, v, create_graph=True)
    dv, = torch.autograd.grad(dx, v, g)
    _check_dropout(g, dv, 0.3, 9)


@pytest.mark.gpu
def test_dropout_seeds_in_a_graph_and_on_another_stream():
    """draw_seed follows torch.manual_seed; a captured call draws a new mask on every replay and its
    backward takes that mask; another stream gives the same bits."""
    torch.manual_seed(5)
    first = adapter.draw_seed("cuda")
    torch.manual_seed(5)
    assert torch.equal(first, adapter.draw_seed("cuda"))
    assert not torch.equal(first, adapter.draw_seed("cuda"))
    x = torch.ones(64, 72, device="cuda", dtype=torch.float16, requires_grad=True)
    want = adapter.dropout(x, 0.4, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = adapter.dropout(x, 0.4, first)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, other)
    static, ones = torch.ones(64, 72, device="cuda").half().requires_grad_(), torch.ones_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = adapter.dropout(static, 0.4, adapter.draw_seed("cuda"))
        dx, = torch.autograd.grad(y, static, ones)
    masks = []
    for _ in range(3):
        graph.replay()
        assert torch.equal(y, dx)
        masks.append(y.detach().clone())
    assert not torch.equal(masks[0], masks[1]) and not torch.equal(masks[1], masks[2])


@pytest.mark.gpu
def test_dropout_past_32_bit_offsets():
    """Elements beyond 2^31 and beyond 2^32: the counter and the addresses are 64 bits wide."""
    cols = 1 << 16
    rows = (1 << 16) + 40
    x = torch.ones(rows, cols, dtype=torch.float16, device="cuda")
    y = adapter.dropout(x, 0.25, _seed(77))
    for row in (0, (1 << 15) - 1, 1 << 15, (1 << 16) - 1, 1 << 16, rows - 1):
        kept, factor = oracle.keep_mask(cols, 0.25, 77, first=row * cols)
        want = torch.from_numpy(np.where(kept, np.float32(factor), 0)).half().cuda()
        assert torch.equal(y[row], want), row


@pytest.mark.gpu
def test_dropout_mask_does_not_depend_on_the_type_or_the_size():
    """One seed's mask over long, odd-sized tensors of each type, and over their first elements."""
    n = 75_000_003
    masks = [adapter.dropout(torch.ones(n, dtype=t, device="cuda"), 0.3, _seed(9)) != 0
             for t in (torch.bfloat16, torch.float16, torch.float32)]
    few = adapter.dropout(torch.ones(100_001, device="cuda").half(), 0.3, _seed(9)) != 0
    assert torch.equal(masks[0], masks[1]) and torch.equal(masks[0], masks[2])
    assert torch.equal(masks[0][:100_001], few)


# ------------------------------------------------------------------------------------------
# the branch
# ------------------------------------------------------------------------------------------
def _branch_inputs(rows, n_in, n_out, rank, seed, g_std=0.05):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std
    a = (torch.rand(rank, n_in, generator=g, device="cuda") * 2 - 1) / math.sqrt(n_in)
    return (normal(rows, n_in).half(), normal(rows, n_out).half(), a,
            normal(n_out, rank, std=0.05), normal(rows, n_out, std=g_std).half())


def _check_branch(x, base, a, b, scaling, p, seed, g, y, dx, da, db):
    host = [t.detach().double().cpu().numpy() for t in (x, base, a, b, g)]
    want, sums = oracle.branch(*host[:4], scaling, p, seed, host[4])
    for name, got, ref, total, half in zip(("y", "dx", "da", "db"), (y, dx, da, db), want, sums,
                                           (1, 1, 0, 0)):
        got = got.detach().double().cpu().numpy()
        if half:
            tol = 2.0 ** -11 * np.abs(ref) + 2.0 ** -25 + 2.0 ** -16 * total
        else:
            tol = 2.0 ** -19 * total + 1e-37
        err = np.abs(got - ref)
        assert (err <= tol).all(), (name, float((err / tol).max()))


def _run_branch(x, base, a, b, scaling, p, seed, g):
    leaves = [t.detach().requires_grad_() for t in (x, base, a, b)]
    y = adapter.lora_branch(*leaves, scaling, p, _seed(seed) if p else None)
    dx, dbase, da, db = torch.autograd.grad(y, leaves, g)
    assert torch.equal(dbase, g)
    return y, dx, da, db


BRANCHES = [(1, 8, 8, 1), (1, 1536, 256, 16), (3, 64, 72, 4), (15, 136, 8, 8), (16, 64, 64, 16),
            (17, 72, 200, 12), (64, 256, 128, 16), (65, 1536, 1536, 16), (130, 320, 264, 33),
            (200, 8960, 1536, 16), (257, 1536, 8960, 64), (1126, 1536, 256, 16),
            (2048, 264, 520, 32), (515, 104, 88, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n_in,n_out,rank", BRANCHES)
def test_branch_matches_the_oracle(rows, n_in, n_out, rank):
    for p in (0.05, 0.0, 0.6):
        inputs = _branch_inputs(rows, n_in, n_out, rank, rows + rank)
        out = _run_branch(*inputs[:4], 2.0, p, 11 + rows, inputs[4])
        _check_branch(*inputs[:4], 2.0, p, 11 + rows, inputs[4], *out)
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_branch_has_dropouts_mask_and_the_formulas_gradient():
    """The branch against dropout + autograd of the plain products in float64, and its gradients
    against differences: y is linear in A, in B and in x, so a central difference of the exact
    branch is exact up to fp64 rounding."""
    x, base, a, b, g = _branch_inputs(48, 96, 80, 16, 3)
    y, dx, da, db = _run_branch(x, base, a, b, 0.5, 0.2, 21, g)
    leaves = [t.double().requires_grad_() for t in (x, a, b)]
    mask = (adapter.dropout(torch.ones_like(x), 0.2, _seed(21)) > 0).double()
    factor = 32768 / (32768 - adapter.drop_threshold(0.2))
    ref = base.double() + 0.5 * (leaves[0] * mask * factor) @ leaves[1].t() @ leaves[2].t()
    grads = torch.autograd.grad(ref, leaves, g.double())
    assert (y.double() - ref).norm() < 2.0 ** -11 * ref.norm()
    assert (dx.double() - grads[0]).norm() < 2.0 ** -11 * grads[0].norm()
    for got, want in ((da, grads[1]), (db, grads[2])):
        assert (got.double() - want).norm() < 2.0 ** -20 * want.norm()

    def loss(xv, av, bv):
        kept, f = oracle.keep_mask(xv.size, 0.2, 21)
        xd = np.where(kept.reshape(xv.shape), xv, 0.0) * f
        return float((g64 * (0.5 * (xd @ av.T) @ bv.T)).sum())
    x64, a64, b64, g64 = (t.double().cpu().numpy() for t in (x, a, b, g))
    rng = np.random.default_rng(0)
    for which, grad in ((0, dx), (1, da), (2, db)):
        args = [x64, a64, b64]
        step = rng.standard_normal(args[which].shape)
        args[which] = args[which] + step
        up = loss(*args)
        args[which] = args[which] - 2 * step
        slope = (up - loss(*args)) / 2
        found = float((grad.double().cpu().numpy() * step).sum())
        scale = float((np.abs(grad.double().cpu().numpy() * step) ** 2).sum()) ** 0.5
        # fp16 gradients are off by 2^-11 of each term at random, fp32 ones far less: six sigma
        assert abs(found - slope) <= 6 * 2.0 ** -11 * scale, which


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [16, 32, 64])
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_branch_of_many_tiles(rank, p):
    """Enough rows that every CTA walks over many tiles and stages of its rings several times, against
    fp64 products on the GPU: relative norms within half a step of fp16 (y, dx) and 2^-20 (dA, dB)."""
    x, base, a, b, g = _branch_inputs(20000, 1032, 1160, rank, 17)
    y, dx, da, db = _run_branch(x, base, a, b, 0.5, p, 33, g)
    mask = adapter.dropout(torch.ones_like(x), p, _seed(33)).bool().double()
    mask *= 32768 / (32768 - adapter.drop_threshold(p))
    a64, b64, g64 = a.double(), b.double(), g.double()
    xd = x.double() * mask
    t, dt = xd @ a64.t(), 0.5 * g64 @ b64
    for got, want, tol in ((y, base.double() + 0.5 * t @ b64.t(), 2.0 ** -11),
                           (dx, (dt @ a64) * mask, 2.0 ** -11), (da, dt.t() @ xd, 2.0 ** -20),
                           (db, 0.5 * g64.t() @ t, 2.0 ** -20)):
        rows = (got.double() - want).norm(dim=1) / want.norm(dim=1).clamp(min=1e-30)
        assert float(rows.max()) < tol, float(rows.max())
    again = _run_branch(x, base, a, b, 0.5, p, 33, g)
    assert all(torch.equal(u, v) for u, v in zip((y, dx, da, db), again))
    assert _lib.device_status() == 0


@pytest.mark.gpu
def test_branch_layouts():
    """Leading dimensions, rows of wider tensors, odd offsets and strides, broadcast gradients, a
    frozen input or adapter."""
    x, base, a, b, g = _branch_inputs(24, 64, 48, 8, 5)
    want = _run_branch(x, base, a, b, 1.0, 0.1, 2, g)
    wide = torch.zeros(24, 83, device="cuda", dtype=torch.float16)
    for at in (0, 3, 8):
        wide[:, at:at + 64] = x
        got = _run_branch(wide[:, at:at + 64], base.t().contiguous().t(), a.t().contiguous().t(), b,
                          1.0, 0.1, 2, g.t().contiguous().t())
        assert all(torch.equal(u, v) for u, v in zip(want, got)), at
    got = _run_branch(x.view(2, 3, 4, 64), base.view(2, 3, 4, 48), a, b, 1.0, 0.1, 2,
                      g.view(2, 3, 4, 48))
    assert all(torch.equal(u, v.view_as(u)) for u, v in zip(want, got))
    leaves = [t.clone().requires_grad_() for t in (x, base, a, b)]
    y = adapter.lora_branch(*leaves, 1.0, 0.1, _seed(2))
    ones = torch.autograd.grad(y.sum(), leaves, retain_graph=True)
    full = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert all(torch.equal(u, v) for u, v in zip(ones, full))
    for frozen in range(4):
        leaves = [t.clone().requires_grad_(i != frozen) for i, t in enumerate((x, base, a, b))]
        y = adapter.lora_branch(*leaves, 1.0, 0.1, _seed(2))
        y.backward(g)
        for i, (leaf, ref) in enumerate(zip(leaves, (want[1], g, want[2], want[3]))):
            assert leaf.grad is None if i == frozen else torch.equal(leaf.grad, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_branch_each_gradient_alone(p):
    """A gradient asked for by itself (another choice of launches) has the bits it has among all."""
    x, base, a, b, g = _branch_inputs(1500, 264, 1032, 12, 6)
    _, *want = _run_branch(x, base, a, b, 1.0, p, 2, g)
    want.insert(1, g)
    for alone in range(4):
        leaves = [t.clone().requires_grad_(i == alone) for i, t in enumerate((x, base, a, b))]
        y = adapter.lora_branch(*leaves, 1.0, p, _seed(2) if p else None)
        got, = torch.autograd.grad(y, leaves[alone], g)
        assert torch.equal(got, want[alone]), alone


@pytest.mark.gpu
def test_branch_of_no_rows():
    x, base, a, b, _ = _branch_inputs(1, 64, 48, 8, 5)
    leaves = [t.clone().requires_grad_() for t in (x[:0], base[:0], a, b)]
    y = adapter.lora_branch(*leaves, 1.0, 0.1, _seed(2))
    assert y.shape == (0, 48)
    y.backward(torch.zeros_like(y))
    assert leaves[0].grad.shape == (0, 64)
    assert not leaves[2].grad.any() and not leaves[3].grad.any()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** -14, 1.0, 2.0 ** 60])
def test_branch_scales(scale):
    """Adapters and gradients far from one: A and B scaled by a power of two and its inverse give
    the same output (their split has to follow their size), and dA, dB scaled the other way;
    rows of very different sizes side by side keep their own precision."""
    x, base, a, b, g = _branch_inputs(80, 128, 96, 16, 8)
    g[::7] *= 2.0 ** -10
    x[::5] *= 2.0 ** -8
    out = _run_branch(x, base, a * scale, b / scale, 2.0, 0.1, 6, g)
    _check_branch(x, base, a * scale, b / scale, 2.0, 0.1, 6, g, *out)


@pytest.mark.gpu
def test_branch_edge_values():
    """B of zeros (a new adapter) leaves base as it is; everything dropped; infinities and NaN in
    dropped places do not come through, those in kept places do, in their own row."""
    x, base, a, b, g = _branch_inputs(40, 64, 48, 8, 5)
    y, dx, da, db = _run_branch(x, base, a, torch.zeros_like(b), 1.0, 0.1, 2, g)
    assert torch.equal(y, base) and not dx.any() and not da.any() and db.any()
    y, dx, da, db = _run_branch(x, base, a, b, 1.0, 1.0, 2, g)
    assert torch.equal(y, base) and not dx.any() and not da.any() and not db.any()
    want = _run_branch(x, base, a, b, 1.0, 0.5, 2, g)
    mask = adapter.dropout(torch.ones_like(x), 0.5, _seed(2)) > 0
    bad = x.clone()
    bad[~mask] = float("nan")
    got = _run_branch(bad, base, a, b, 1.0, 0.5, 2, g)
    assert all(torch.equal(u, v) for u, v in zip(want, got))
    bad = x.clone()
    row = 17
    bad[row, mask[row].nonzero()[0, 0]] = float("inf")
    y = _run_branch(bad, base, a, b, 1.0, 0.5, 2, g)[0]
    assert not torch.isfinite(y[row]).all()
    keep = torch.arange(40, device="cuda") != row
    assert torch.equal(y[keep], want[0][keep])


@pytest.mark.gpu
def test_branch_same_bits_on_streams_and_in_graphs():
    """The same bits twice, on another stream, and in two captured graphs replayed in turn (each
    has its own workspace)."""
    x, base, a, b, g = _branch_inputs(300, 520, 264, 16, 12)
    want = _run_branch(x, base, a, b, 2.0, 0.1, 31, g)
    again = _run_branch(x, base, a, b, 2.0, 0.1, 31, g)
    assert all(torch.equal(u, v) for u, v in zip(want, again))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _run_branch(x, base, a, b, 2.0, 0.1, 31, g)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(want, other))
    seed = _seed(31)
    graphs = []
    for _ in range(2):
        leaves = [t.clone().requires_grad_() for t in (x, base, a, b)]
        gs = g.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = adapter.lora_branch(*leaves, 2.0, 0.1, seed)
            grads = torch.autograd.grad(y, (leaves[0], leaves[2], leaves[3]), gs)
        graphs.append((graph, leaves, y, grads))
    with torch.no_grad():
        graphs[1][1][0].mul_(0.5)
    for _ in range(2):
        for graph, *_ in graphs:
            graph.replay()
    assert all(torch.equal(u, v) for u, v in zip(want, (graphs[0][2], *graphs[0][3])))
    half = _run_branch(x * 0.5, base, a, b, 2.0, 0.1, 31, g)
    assert all(torch.equal(u, v) for u, v in zip(half, (graphs[1][2], *graphs[1][3])))


@pytest.mark.gpu
def test_branch_saves_its_input_and_rank_wide_operands_only():
    """What a call keeps for its backward: x as it is (changing it in place is an error, as is
    changing the seed), the rank-wide parts, no mask and no dropped copy; nothing without grad."""
    x, base, a, b, g = _branch_inputs(4096, 1536, 64, 16, 3)
    a.requires_grad_()
    b.requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        y = adapter.lora_branch(x, base, a, b, 1.0, 0.1, _seed(1))
    assert y.grad_fn is None
    assert torch.cuda.memory_allocated() - before <= y.numel() * 2 + 4096
    del y
    seed = _seed(1)
    before = torch.cuda.memory_allocated()
    y = adapter.lora_branch(x, base, a, b, 1.0, 0.1, seed)
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    # t's parts (128 bytes a row), the parts of A and B for the backward pass
    assert kept <= 4096 * 128 + 16 * 2 * 2 * 64 + 1536 * 128 + (1 << 15) < x.numel() // 8
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward(g)
    y = adapter.lora_branch(x, base, a, b, 1.0, 0.1, _seed(1))
    x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward(g)


@pytest.mark.gpu
def test_branch_past_32_bit_offsets():
    """Rows whose elements lie beyond 2^32: their masks and products, forward and backward."""
    cols, rank = 8960, 4
    rows = (1 << 32) // cols + 200
    g = torch.Generator("cuda").manual_seed(2)
    x = torch.empty(rows, cols, dtype=torch.float16, device="cuda")
    x[:1000].normal_(generator=g)
    at = [0, 1, rows - 150, rows - 1]
    for i in at:
        x[i].normal_(generator=g)
    x[1000:rows - 200] = 0
    x[rows - 200:].normal_(generator=g)
    base = torch.zeros(rows, 8, dtype=torch.float16, device="cuda")
    a = (torch.rand(rank, cols, generator=g, device="cuda") - 0.5) * 0.02
    b = torch.randn(8, rank, generator=g, device="cuda")
    dy = torch.randn(rows, 8, generator=g, device="cuda").half()
    x.requires_grad_()
    y = adapter.lora_branch(x, base, a, b, 1.0, 0.3, _seed(8))
    dx, = torch.autograd.grad(y, x, dy)
    for i in at:
        kept, factor = oracle.keep_mask(cols, 0.3, 8, first=i * cols)
        m = torch.from_numpy(kept).cuda().double() * factor
        want = ((x[i].double() * m) @ a.double().t()) @ b.double().t()
        scale = ((x[i].double() * m).abs() @ a.double().abs().t()) @ b.double().abs().t()
        assert ((y[i].double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -16 * scale).all()
        want = (dy[i].double() @ b.double() @ a.double()) * m
        scale = (dy[i].double().abs() @ b.double().abs() @ a.double().abs()) * m
        err = (dx[i].double() - want).abs()
        assert (err <= 2.0 ** -11 * want.abs() + 2.0 ** -25 + 2.0 ** -16 * scale).all()


@pytest.mark.gpu
def test_branches_on_two_streams_at_once():
    """Calls that overlap on the GPU: each has workspaces of its own."""
    cases = [_branch_inputs(1500, 1536, 520, 16, 4), _branch_inputs(900, 520, 1536, 64, 5)]
    want = [_run_branch(*c[:4], 1.0, 0.2, 3, c[4]) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (c, stream) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(stream):
                got[i].append(_run_branch(*c[:4], 1.0, 0.2, 3, c[4]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(u, v) for u, v in zip(want[i], out))
    assert _lib.device_status() == 0


# ------------------------------------------------------------------------------------------
# the branch in its module and in the training step
# ------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_branch_captured_behind_copies_and_joined_streams():
    """Captured behind a copy (a node that is no kernel) and behind two streams that have been
    joined (two nodes), forward and backward apart on their own graphs' inputs."""
    x, base, a, b, g = _branch_inputs(140, 136, 264, 8, 21)
    want = _run_branch(x, base, a, b, 2.0, 0.1, 31, g)
    seed = _seed(31)
    leaves = [torch.zeros_like(t).requires_grad_() for t in (x, base, a, b)]
    gs, doubled = torch.zeros_like(g), torch.zeros_like(g)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        with torch.no_grad():
            for t, v in zip(leaves, (x, base, a, b)):
                t.copy_(v)
            with torch.cuda.stream(side):
                gs.copy_(g)
        torch.cuda.current_stream().wait_stream(side)
        y = adapter.lora_branch(*leaves, 2.0, 0.1, seed)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            doubled.copy_(gs).mul_(2)
        torch.cuda.current_stream().wait_stream(side)
        grads = torch.autograd.grad(y, (leaves[0], leaves[2], leaves[3]), gs)
        after = y.detach().clone()
    for _ in range(2):
        graph.replay()
    assert all(torch.equal(u, v) for u, v in zip(want, (after, *grads)))
    assert torch.equal(doubled, 2 * g)


@pytest.mark.gpu
def test_branch_that_drops_everything():
    x, base, a, b, g = _branch_inputs(70, 136, 72, 8, 22)
    x[3, 5] = float("inf")
    y, dx, da, db = _run_branch(x, base, a, b, 2.0, 1.0, 31, g)
    assert torch.equal(y, base) and not dx.any() and not da.any() and not db.any()


TINY = dict(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
            num_attention_heads=8, num_key_value_heads=2)


@pytest.mark.gpu
def test_fused_module_and_its_unfused_way_share_their_mask():
    """A rank beyond the branch's and another type go through `dropout` and stock products: the
    same mask for the same torch seed, results equal up to those products' fp16 roundings."""
    model = qlora.build_model(qlora.qwen25_15b_config(**TINY), "cuda", lora_fused=True,
                              lora_dropout=0.3, lora_b_std=0.05)
    module = model.model.layers[0].self_attn.q_proj
    module.train()
    x = torch.randn(40, 512, device="cuda").half()

    def call(v, m=module):
        model.model.layers[0]._talm_layer_group.start_forward()
        torch.manual_seed(3)
        return m(v)
    fused = call(x)
    other = call(x.float())
    assert other.dtype == torch.float32
    torch.testing.assert_close(other.half(), fused, rtol=2e-3, atol=2e-3)
    wide = qlora.LoraLinear(module.base, 80, 160, 0.3, b_std=0.05, fused=True).train()
    with torch.no_grad():
        wide.lora_A[:16].copy_(module.lora_A)
        wide.lora_B.zero_()
        wide.lora_B[:, :16].copy_(module.lora_B)
    torch.testing.assert_close(call(x, wide), fused, rtol=2e-3, atol=2e-3)
    module.eval()
    quiet = call(x)
    assert torch.equal(quiet, call(x))


@pytest.mark.gpu
def test_adapters_cast_to_fp16_keep_working():
    """model.half() makes the adapters fp16, which the kernels do not take: the fused module and the
    served one go through the stock products and give what those give."""
    model = qlora.build_model(qlora.qwen25_15b_config(**TINY), "cuda", lora_fused=True, seed=5,
                              lora_dropout=0.0, lora_b_std=0.05)
    layer = model.model.layers[0]
    module = layer.self_attn.q_proj
    module.lora_A.data, module.lora_B.data = module.lora_A.data.half(), module.lora_B.data.half()
    x = torch.randn(4, 512, device="cuda").half()

    def call():
        layer._talm_layer_group.start_forward()
        return module(x)
    got = call()
    module.fused = False
    want = call()
    assert torch.equal(got, want)
    with torch.no_grad(), qgroup.serving():
        served = call()
    # the base's weights rounded or not: 2^-11 of each term, and of the result
    assert (served.float() - want.float()).norm() < 2e-3 * want.float().norm()


@pytest.mark.gpu
def test_training_step_with_fused_adapters():
    """The model with fused adapters against the stock ones on the same batch without dropout:
    losses within 1e-3 and adapter gradients within 2e-2 in norm (fp16 roundings of the stock
    adapter's products); with dropout, the eager step twice from one torch seed gives the same
    gradients, and gradient checkpointing, which runs the forward again, the same loss."""
    config = qlora.qwen25_15b_config(**TINY)
    kw = dict(seed=7, lora_dropout=0.0, lora_b_std=0.02)
    stock = qlora.build_model(config, "cuda", **kw)
    fused = qlora.build_model(config, "cuda", lora_fused=True, **kw)
    qlora.patch()
    batch = qlora.make_batch(4, 128, TINY["vocab_size"], "cuda", seed=1)
    grads, losses = [], []
    for model in (stock, fused):
        model.train()
        out = model(**batch)
        out.loss.backward()
        losses.append(out.loss.detach())
        grads.append({n: p.grad for n, p in model.named_parameters() if p.requires_grad})
    torch.testing.assert_close(losses[1], losses[0], rtol=1e-3, atol=0)
    for name in grads[0]:
        err = (grads[1][name] - grads[0][name]).norm() / grads[0][name].norm().clamp(min=1e-30)
        assert float(err) < 2e-2, (name, float(err))
    model = qlora.build_model(config, "cuda", lora_fused=True, seed=7, lora_dropout=0.2,
                              lora_b_std=0.02)
    model.train()
    results = []
    for checkpointed in (False, False, True):
        if checkpointed:
            model.gradient_checkpointing_enable({"use_reentrant": False})
        model.zero_grad(set_to_none=True)
        torch.manual_seed(11)
        loss = model(**batch).loss
        loss.backward()
        results.append((loss.detach(), [p.grad.clone() for p in qlora.adapters(model)]))
    assert torch.equal(results[0][0], results[1][0])
    assert all(torch.equal(u, v) for u, v in zip(results[0][1], results[1][1]))
    torch.testing.assert_close(results[2][0], results[0][0], rtol=1e-5, atol=0)
    for u, v in zip(results[0][1], results[2][1]):
        assert (u - v).norm() <= 1e-3 * u.norm()


@pytest.mark.gpu
def test_graphed_step_with_fused_adapters():
    """The decoder's forward and backward as CUDA graphs: without dropout the eager step's losses
    over three steps, with dropout a new mask on every replay (another loss at a rate of zero)."""
    config = qlora.qwen25_15b_config(**TINY)
    batch = qlora.make_batch(4, 128, TINY["vocab_size"], "cuda", seed=5)
    n_lab = qlora.labelled_count(batch["labels"])
    qlora.patch()
    kw = dict(seed=11, lora_dropout=0.0, lora_b_std=0.02, lora_fused=True)
    eager, graphed = (qlora.build_model(config, "cuda", **kw).train() for _ in range(2))
    opts = [torch.optim.AdamW(qlora.adapters(m), lr=1e-3) for m in (eager, graphed)]
    step = qlora.GraphedStep(graphed, opts[1], batch)
    for _ in range(3):
        a = qlora.train_step(eager, opts[0], batch)
        torch.testing.assert_close(step(batch, n_lab), a, rtol=1e-5, atol=0)
    kw.update(lora_dropout=0.5, lora_b_std=0.2)
    model = qlora.build_model(config, "cuda", **kw).train()
    step = qlora.GraphedStep(model, torch.optim.SGD(qlora.adapters(model), lr=0.0), batch)
    losses = {float(step(batch, n_lab)) for _ in range(4)}
    assert len(losses) == 4 and all(math.isfinite(v) for v in losses)


@pytest.mark.gpu
def test_adapted_projection_trains_and_serves():
    """One adapted 4-bit projection, as it is used: trained through the fused branch, then served
    token by token; both forms give the same output up to fp16 roundings of the weights."""
    model = qlora.build_model(qlora.qwen25_15b_config(**TINY), "cuda", lora_fused=True, seed=3,
                              lora_dropout=0.1, lora_b_std=0.05)
    layer = model.model.layers[0]
    module = layer.self_attn.q_proj
    assert isinstance(module.base, nf4_format.NF4Linear)
    x = torch.randn(20, 512, device="cuda").half().requires_grad_()
    module.train()
    opt = torch.optim.SGD([module.lora_A, module.lora_B], lr=0.5)
    for _ in range(2):
        layer._talm_layer_group.start_forward()
        opt.zero_grad()
        module(x).float().square().mean().backward()
        opt.step()
    module.eval()
    with torch.no_grad():
        layer._talm_layer_group.start_forward()
        whole = module(x)
        with qgroup.serving(1):
            served = torch.cat([module(x[i:i + 1]) for i in range(20)])
    assert (served.float() - whole.float()).norm() < 2e-3 * whole.float().norm()
