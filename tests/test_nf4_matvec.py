"""The few-row NF4 product (with its adapter) against a float64 oracle.

Error bounds, from the arithmetic: the result is rounded to fp16 once (at most 2^-11 of it, 2^-25 below
the normal range). The kernel holds the 16 levels in fp16 after scaling them by a constant that makes
their rounding small (relative errors of 6.2e-5 in the mean square over the levels, 2.9e-4 at most);
over one output these are independent, so six standard deviations of the sum are
6 * 6.2e-5 * |w o x|, with 1.5 more for the levels' unequal shares in a short row. fp32 products
and sums of a row's terms add 2^-20 of the sum of their magnitudes."""

import math

import numpy as np
import pytest
import torch

from oracle import adapter as oracle
from talm_b200 import _lib, build, nf4_dequant, qgroup, qlora

LEVEL_RMS, LEVEL_MAX = 6.2e-5, 2.9e-4


def _bound(w, x, y, extra):
    """[rows, out] bound of |got - y| (see the module's docstring)."""
    terms = np.sqrt((x ** 2) @ (w ** 2).T)
    total = np.abs(x) @ np.abs(w).T
    level = np.minimum(6 * 1.5 * LEVEL_RMS * terms, LEVEL_MAX * total)
    return 2.0 ** -11 * np.abs(y) + 2.0 ** -25 + level + 2.0 ** -20 * (total + extra)


class _Case:
    """Random arrays of one product on the device, and its float64 result."""

    def __init__(self, rows, n_out, n_in, form, seed, block=64, qblock2=256, row0=0, bias=False,
                 rank=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        n = n_out * n_in
        blocks = -(-n // block)
        self.n_out, self.n_in, self.block, self.qblock2, self.row0 = n_out, n_in, block, qblock2, row0
        x = torch.randn(rows, n_in, generator=g).half()
        self.packed = torch.randint(0, 256, (n // 2,), generator=g, dtype=torch.uint8)
        self.bias = (torch.randn(n_out, generator=g) * 0.1).half() if bias else None
        if form == "absmax":
            self.absmax = torch.rand(blocks, generator=g) * 0.05 + 0.01
            scales = self.absmax.numpy()
        else:
            self.absmax8 = torch.randint(0, 256, (blocks,), generator=g, dtype=torch.uint8)
            self.code = torch.sort(torch.rand(256, generator=g) * 2 - 1).values
            n2 = -(-(row0 + blocks) // qblock2)
            self.absmax2 = torch.rand(n2, generator=g) * 0.01
            self.offset2 = torch.rand(n2, generator=g) * 0.03
            scales = oracle.double_quant_scales(self.absmax8.numpy(), self.code.numpy(),
                                                self.absmax2.numpy(), self.offset2.numpy(), row0,
                                                qblock2)
        w = oracle.nf4_weight(self.packed.numpy(), scales, n_out, n_in, block)
        x64 = x.double().numpy()
        y = x64 @ w.T
        extra = 0.0
        self.adapter = None
        if rank:
            a = (torch.rand(rank, n_in, generator=g) * 2 - 1) / math.sqrt(n_in)
            b = torch.randn(n_out, rank, generator=g) * 0.1
            a64, b64 = a.double().numpy(), b.double().numpy()
            y = y + 1.5 * (x64 @ a64.T) @ b64.T
            extra = 1.5 * (np.abs(x64) @ np.abs(a64).T) @ np.abs(b64).T
            self.adapter = (a.to(device), b.to(device), 1.5)
        if bias:
            y = y + self.bias.double().numpy()
            extra = extra + np.abs(self.bias.double().numpy())
        self.y, self.tol = y, _bound(w, x64, y, extra)
        self.x = x.to(device)
        for name in ("packed", "bias", "absmax", "absmax8", "code", "absmax2", "offset2"):
            t = getattr(self, name, None)
            if t is not None:
                setattr(self, name, t.to(device))
        self.levels = torch.tensor(qgroup.NF4_LEVELS, device=device)
        self.form = form

    def run(self, x=None, out=None, rows=None):
        x = self.x if x is None else x
        if self.form == "absmax":
            return nf4_dequant.nf4_matvec(x, self.packed, self.absmax, self.block, out=out,
                                          bias=self.bias, adapter=self.adapter)
        if out is None:
            out = torch.empty(x.reshape(-1, self.n_in).shape[0], self.n_out, dtype=torch.float16,
                              device=x.device)
        return qgroup.launch_matvec(x, self.packed, self.absmax8, self.code, self.absmax2,
                                    self.offset2, self.levels, out, self.row0, self.n_out,
                                    self.n_in, self.block, self.qblock2, bias=self.bias,
                                    adapter=self.adapter)

    def check(self, got):
        err = np.abs(got.double().cpu().numpy() - self.y)
        assert (err <= self.tol).all(), float((err / self.tol).max())


# ------------------------------------------------------------------------------------------
# refusals, before any launch
# ------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_c_entry_rejects_bad_arguments(lib):
    def call(n_rows=1, w_rows=8, w_cols=64, block=64, qblock2=256, rank=0, ld_x=64, ld_y=8,
             absmax8=None, row0=0):
        return lib.talm_nf4_matvec(None, ld_x, n_rows, None, absmax8, None, None, None, None, None,
                                   row0, w_rows, w_cols, block, qblock2, None, None, None, rank,
                                   1.0, None, None, ld_y, None)
    assert call(n_rows=33) == 1 and call(n_rows=-1) == 1
    assert call(w_cols=63) == 1 and call(w_cols=0) == 1 and call(w_rows=-1) == 1
    assert call(block=63) == 1 and call(block=0) == 1
    assert call(absmax8=16, qblock2=0) == 1 and call(absmax8=16, row0=-1) == 1
    assert call(rank=65) == 1 and call(rank=-1) == 1
    assert call(ld_x=63) == 1 and call(ld_y=7) == 1
    assert call(w_rows=1 << 20, w_cols=1 << 22, ld_x=1 << 22, ld_y=1 << 20) == 3
    assert call() == 1 and b"null" in lib.talm_last_error()
    assert call(n_rows=0) == 0 and call(w_rows=0) == 0


def test_python_entries_refuse_what_the_kernel_does_not_take():
    c = _Case(2, 8, 64, "group", 0, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        c.run()
    with pytest.raises(TypeError, match="fp16"):
        c.run(c.x.float())
    with pytest.raises(ValueError, match="at most 32"):
        c.run(torch.zeros(33, 64, dtype=torch.float16))
    with pytest.raises(ValueError, match="last dimension"):
        c.run(torch.zeros(2, 32, dtype=torch.float16))
    with pytest.raises(ValueError, match="shorter"):
        qgroup.launch_matvec(c.x, c.packed[1:], c.absmax8, c.code, c.absmax2, c.offset2, c.levels,
                             torch.empty(2, 8).half(), 0, 8, 64, 64, 256)
    with pytest.raises(ValueError, match="shorter"):  # the second level ends before the last block
        qgroup.launch_matvec(c.x, c.packed, c.absmax8, c.code, c.absmax2, c.offset2, c.levels,
                             torch.empty(2, 8).half(), 256, 8, 64, 64, 256)
    with pytest.raises(ValueError, match="out must be"):
        c.run(out=torch.empty(2, 9).half())
    for row0, block, block2 in ((0, 0, 256), (0, 64, 0), (-1, 64, 256)):
        with pytest.raises(ValueError, match="positive"):
            qgroup.launch_matvec(c.x, c.packed, c.absmax8, c.code, c.absmax2, c.offset2, c.levels,
                                 torch.empty(2, 8).half(), row0, 8, 64, block, block2)
    d = _Case(2, 8, 64, "absmax", 0, device="cpu")
    with pytest.raises(ValueError, match="scales for"):
        nf4_dequant.nf4_matvec(d.x, d.packed, d.absmax[:-1], 64)
    with pytest.raises(ValueError, match="rows of"):
        nf4_dequant.nf4_matvec(torch.zeros(1, 60, dtype=torch.float16), d.packed, d.absmax, 64)
    with pytest.raises(ValueError, match="does not map"):
        nf4_dequant.nf4_matvec(d.x, d.packed, d.absmax, 64,
                               adapter=(torch.zeros(4, 32), torch.zeros(8, 4), 1.0))
    with pytest.raises(ValueError, match="0..32"):
        with qgroup.serving(33):
            pass


def test_serving_is_scoped_and_left_alone_by_gradients_and_cpu_tensors():
    x = torch.zeros(1, 64, dtype=torch.float16)
    assert not qgroup.takes_matvec(x)
    with qgroup.serving(4):
        with torch.no_grad():
            assert not qgroup.takes_matvec(x)  # a CPU tensor keeps its path
        with qgroup.serving(0):
            assert qgroup._SERVING["rows"] == 0
        assert qgroup._SERVING["rows"] == 4
    assert qgroup._SERVING["rows"] == 0


# ------------------------------------------------------------------------------------------
# the kernel
# ------------------------------------------------------------------------------------------
SHAPES = [(1, 64), (16, 64), (17, 128), (5, 192), (256, 1536), (1001, 2112), (40, 8960),
          (2053, 320),           # whole 64-column blocks
          (3, 2), (33, 50), (7, 96), (130, 1000)]  # rows that blocks straddle


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["group", "absmax"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 32])
def test_matches_the_oracle(rows, shape, form):
    bias = (rows + shape[0]) % 2 == 0
    c = _Case(rows, *shape, form, seed=rows * 131 + shape[1], bias=bias, row0=7, qblock2=3)
    c.check(c.run())
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 9, 32])
@pytest.mark.parametrize("shape", [(60011, 64), (40000, 192), (17920, 1536)],
                         ids=lambda s: f"{s[0]}x{s[1]}")
def test_many_tiles(shape, rows):
    """More tiles than the GPU's warps: every warp walks over several, its ring many times around."""
    for form, rank in (("group", 0), ("absmax", 16)):
        c = _Case(rows, *shape, form, seed=rows + shape[1], bias=True, rank=rank, block=64, row0=5)
        c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("block", [2, 6, 64, 96, 128, 256, 4096])
@pytest.mark.parametrize("n_in", [64, 192, 250])
def test_block_sizes(block, n_in):
    for form, qblock2 in (("absmax", 1), ("group", 256), ("group", 5)):
        c = _Case(3, 45, n_in, form, seed=block + n_in, block=block, qblock2=qblock2, row0=11)
        c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [1, 3, 8, 16, 33, 64])
@pytest.mark.parametrize("rows,n_out,n_in", [(1, 256, 1536), (5, 77, 64), (32, 130, 8960),
                                             (9, 20, 50)])
def test_adapter_in_the_epilogue(rows, n_out, n_in, rank):
    for form in ("group", "absmax"):
        c = _Case(rows, n_out, n_in, form, seed=rank + n_out, bias=rank % 2 == 0, rank=rank)
        c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("n_in", [1024, 2560, 3584, 4096, 5120, 6144, 7168, 8192, 14336])
def test_adapter_widths(n_in):
    """One to eight CTAs share the columns of x A^T."""
    for rows in (1, 20):
        c = _Case(rows, 48, n_in, "group", seed=n_in, rank=24)
        c.check(c.run())


@pytest.mark.gpu
def test_strides_alignment_and_untouched_neighbours():
    """Rows of a wider tensor, an odd storage offset of x, packed bytes and out; what lies between
    the output's rows stays as it was."""
    for n_in in (128, 90):
        c = _Case(6, 37, n_in, "group", seed=n_in, bias=True)
        wide = torch.full((6, n_in + 13), 7.0, dtype=torch.float16, device="cuda")
        wide[:, 5:5 + n_in] = c.x
        out = torch.full((6, 51), -3.0, dtype=torch.float16, device="cuda")
        c.run(wide[:, 5:5 + n_in], out[:, 3:40])
        c.check(out[:, 3:40])
        assert (out[:, :3] == -3).all() and (out[:, 40:] == -3).all()
        moved = torch.empty(c.packed.numel() + 3, dtype=torch.uint8, device="cuda")[3:]
        c.packed = moved.copy_(c.packed)
        c.check(c.run(c.x.t().contiguous().t()))  # columns first
        c.x = c.x[:1].expand(6, n_in)             # one row broadcast
        got = c.run()
        assert torch.equal(got, got[:1].expand_as(got))


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [16, 8, 4, 1])
def test_packed_bytes_on_any_boundary(offset):
    """The wide copies want rows on 16-byte boundaries; weights that start elsewhere (behind an odd
    one in the same buffer) take the other kernel."""
    for rows, shape in ((1, (37, 128)), (9, (256, 1536))):
        c = _Case(rows, *shape, "group", seed=offset, bias=True, rank=8)
        whole = torch.empty(c.packed.numel() + 32, dtype=torch.uint8, device="cuda")
        assert whole.data_ptr() % 16 == 0
        moved = whole[offset:offset + c.packed.numel()]
        c.packed = moved.copy_(c.packed)
        c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 9])
def test_extreme_values(rows):
    """Zero scales, an input of zeros, the largest fp16 inputs (an infinite result where the sum
    passes fp16's range), and infinities and NaN, which stay in their own rows."""
    c = _Case(rows, 24, 128, "absmax", seed=rows)
    c.absmax.zero_()
    assert not c.run().any()
    c = _Case(rows, 24, 128, "absmax", seed=rows)
    c.x.zero_()
    assert not c.run().any()
    c = _Case(rows, 24, 128, "absmax", seed=rows)
    c.absmax.fill_(1.0)
    c.packed.fill_(0xFF)
    c.x.fill_(65504.0)
    assert torch.isinf(c.run()).all()
    c.packed.fill_(0xF0)  # +1 and -1 in turn: the sums cancel exactly
    assert not c.run().any()
    c.x[0, 3] = float("inf")
    c.x[-1, 5] = float("nan")
    got = c.run()
    assert torch.isnan(got[-1]).all()
    if rows > 1:
        assert torch.isinf(got[0]).all() and not got[1:-1].any()


@pytest.mark.gpu
def test_one_code_everywhere_keeps_the_levels_error():
    """All weights the same level and all inputs of one sign: the errors of the rounded levels add
    up, and stay under the largest one."""
    for code in range(16):
        c = _Case(1, 8, 256, "absmax", seed=1)
        c.packed.fill_(code * 17)
        c.x.fill_(0.5)
        w = qgroup.NF4_LEVELS[code] * c.absmax.double().view(8, 4).repeat_interleave(64, 1)
        want = (w * 0.5).sum(1)
        err = (c.run().double()[0] - want).abs()
        assert (err <= (LEVEL_MAX + 2.0 ** -11 + 2.0 ** -20) * want.abs()).all(), code


@pytest.mark.gpu
def test_same_bits_every_time_on_any_stream_and_in_a_graph():
    c = _Case(13, 200, 1536, "group", seed=3, bias=True, rank=16)
    first = c.run()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        second = c.run()
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(first, second)
    x, outs = c.x.clone(), []
    graphs = []
    for _ in range(2):  # two captured calls, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        out = torch.empty_like(first)
        with torch.cuda.graph(graph):
            c.run(x, out)
        graphs.append(graph)
        outs.append(out)
    x.copy_(c.x.flip(0))
    for graph in graphs:
        graph.replay()
    want = c.run(x)
    assert all(torch.equal(o, want) for o in outs)
    c.check(want.flip(0))


TINY = dict(vocab_size=500, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
            num_attention_heads=8, num_key_value_heads=2)


@pytest.mark.gpu
@pytest.mark.parametrize("last", [None, 1, 3])
def test_group_spans(last):
    """matvec on the projections of a layer group against the group's dequantised weights."""
    model = qlora.build_model(qlora.qwen25_15b_config(**TINY), "cuda", seed=4)
    group = model.model.layers[1]._talm_layer_group
    first = 0 if last else 5
    stop = last or 6
    x = torch.randn(3, 2, group.shapes[first][1], device="cuda").half()
    got = qgroup.matvec(x, group, first, last)
    w = torch.cat([group.dequantize_one(i) for i in range(first, stop)]).double()
    want = x.double() @ w.t()
    # the dequantised weights are rounded to fp16: 2^-11 of each term, independent (6 sigma)
    terms = (x.double() ** 2 @ (w ** 2).t()).sqrt()
    err = (got.double() - want).abs()
    assert got.shape == (3, 2, w.shape[0])
    assert (err <= 2.0 ** -11 * want.abs() + 6 * (1.5 * LEVEL_RMS + 2.0 ** -11) * terms).all()


@pytest.mark.gpu
@pytest.mark.parametrize("targets", [qlora.LORA_TARGETS, ("mlp.down_proj", "self_attn.q_proj")])
def test_served_model_decodes_like_the_whole_forward(targets):
    """The model token by token with a cache under `serving` against its own whole forward without
    it: the same hidden states up to fp16 (every product of the second is made of weights rounded
    to fp16: 2^-11 per term and layer, far under the 2e-2 asked), the adapters' branches in both;
    `generate` takes the argmax of those logits; outside `serving` nothing has changed."""
    from talm_b200.engaged import RAN

    model = qlora.build_model(qlora.qwen25_15b_config(**TINY), "cuda", seed=6, lora_b_std=0.05,
                              lora_targets=targets)
    qlora.patch()
    model.eval()
    ids = torch.randint(0, TINY["vocab_size"], (2, 9), device="cuda",
                        generator=torch.Generator("cuda").manual_seed(1))
    with torch.no_grad():
        whole = model(input_ids=ids).logits
        before = RAN["matvec"]
        cache, steps = None, []
        with qgroup.serving():
            for i in range(ids.shape[1]):
                out = model(input_ids=ids[:, i:i + 1], past_key_values=cache, use_cache=True)
                cache = out.past_key_values
                steps.append(out.logits)
        assert RAN["matvec"] - before == 9 * 7 * TINY["num_hidden_layers"]
        again = model(input_ids=ids).logits
    assert torch.equal(whole, again)
    stepped = torch.cat(steps, 1).float()
    assert (stepped - whole.float()).norm() < 2e-2 * whole.float().norm()
    model.train()
    text = qlora.generate(model, ids, 5)
    assert model.training and text.shape == (2, 14) and torch.equal(text[:, :9], ids)
    model.eval()
    with torch.no_grad():
        logits = model(input_ids=text[:, :-1]).logits[:, 8:].float()
    chosen = logits.gather(-1, text[:, 9:, None])[..., 0]
    assert (logits.max(-1).values - chosen <= 4e-2 * logits.abs().amax(-1)).all()
