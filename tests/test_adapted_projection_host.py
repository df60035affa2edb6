"""Host side of the adapted 4-bit projections, on CPU tensors (no kernel launches): who is served, what
is refused, what a call leaves behind."""

import os
import re
import threading
from types import SimpleNamespace

import pytest
import torch

from talm_b200 import _lib, adapter, nf4_dequant, nf4_format, qgroup, qlora, state


def _served(rows=1):
    """Whether a CUDA tensor of that many rows would be served now."""
    x = SimpleNamespace(is_cuda=True, shape=(rows, 64), numel=lambda: rows * 64)
    with torch.no_grad():
        return qgroup.takes_matvec(x)


# ------------------------------------------------------------------------------------------
# serving
# ------------------------------------------------------------------------------------------
def test_serving_of_two_threads_that_overlap():
    """A enters, B enters, A leaves, B leaves: each has its own route until it leaves, and nothing stays
    on behind them."""
    turn = [threading.Event() for _ in range(4)]
    seen = {}

    def first():
        with qgroup.serving(4):
            seen["a"] = (_served(4), _served(5))
            turn[0].set()
            turn[1].wait(30)
        seen["a left"] = _served()
        turn[2].set()

    def second():
        turn[0].wait(30)
        seen["b before"] = _served()
        with qgroup.serving(8):
            turn[1].set()
            turn[2].wait(30)
            seen["b"] = (_served(8), _served(9))
        seen["b left"] = _served()

    threads = [threading.Thread(target=f) for f in (first, second)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert seen == {"a": (True, False), "a left": False, "b before": False, "b": (True, False),
                    "b left": False}
    assert not _served()


def test_serving_blocks_that_end_out_of_order():
    """Two blocks of one thread, left in the order in which they were entered."""
    outer, inner = qgroup.serving(4), qgroup.serving(8)
    outer.__enter__()
    inner.__enter__()
    assert _served(8)
    outer.__exit__(None, None, None)
    assert _served(8)
    inner.__exit__(None, None, None)
    assert not _served()


# ------------------------------------------------------------------------------------------
# an adapted projection under serving
# ------------------------------------------------------------------------------------------
@pytest.fixture
def served(monkeypatch):
    """An adapted projection whose few-row product is a dense one on the CPU; `.calls` holds the
    adapters it was given."""
    g = torch.Generator().manual_seed(0)
    w = torch.randn(8, 64, generator=g).half()
    calls = []

    def matvec(x, group, first, last=None, bias=None, adapter=None):
        calls.append(adapter)
        y = x.float() @ w.float().t()
        if adapter is not None:
            y = y + adapter[2] * (x.float() @ adapter[0].t()) @ adapter[1].t()
        return y.half()

    monkeypatch.setattr(qgroup, "matvec", matvec)
    monkeypatch.setattr(qgroup, "takes_matvec", lambda x: not torch.is_grad_enabled())
    base = nf4_format.NF4Linear(torch.zeros(8 * 32, dtype=torch.uint8),
                                SimpleNamespace(shape=(8, 64)))
    base._talm_group = (SimpleNamespace(biases=[None]), 0)
    module = qlora.LoraLinear(base, 4, 8, 0.0, generator=g, b_std=0.1).eval()
    module.calls = calls
    return module


def _call(module, x):
    with torch.no_grad():
        return module(x)


def test_served_projection_is_one_product(served):
    x = torch.randn(2, 64).half()
    _call(served, x)
    assert len(served.calls) == 1 and served.calls[0] is not None


@pytest.mark.parametrize("kind", ["forward", "pre", "global", "global pre", "instance"])
def test_served_projection_runs_the_base_hooks(served, kind):
    """Hooks of the base projection see its call and its result, and what they return counts."""
    x = torch.randn(2, 64).half()
    seen = []
    branch = _call(served, x).float()
    base = served.base
    calls = torch.nn.modules.module
    if kind == "forward":
        handle = base.register_forward_hook(lambda m, a, out: (seen.append(m), out * 0)[1])
    elif kind == "pre":
        handle = base.register_forward_pre_hook(lambda m, a: (seen.append(m), (a[0] * 0,))[1])
    elif kind == "global":
        handle = calls.register_module_forward_hook(
            lambda m, a, out: (seen.append(m), out * 0)[1] if m is base else None)
    elif kind == "global pre":
        handle = calls.register_module_forward_pre_hook(
            lambda m, a: (seen.append(m), (a[0] * 0,))[1] if m is base else None)
    else:
        forward = base.forward
        base.forward = lambda v: (seen.append(base), forward(v) * 0)[1]
        handle = SimpleNamespace(remove=lambda: base.__dict__.pop("forward"))
    try:
        got = _call(served, x).float()
    finally:
        handle.remove()
    want = served.scaling * (x.float() @ served.lora_A.t()) @ served.lora_B.t()
    assert seen == [base]
    assert served.calls[-1] is None  # the base alone: the branch is added to what the hook returned
    assert (got - want).norm() < 1e-2 * want.norm() < branch.norm()
    _call(served, x)
    assert served.calls[-1] is not None


# ------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("which", ["x", "bias", "lora_A", "lora_B", "out"])
def test_few_row_product_refuses_what_asks_for_a_gradient(which):
    """A result without a graph would pass the gradient by: refused where one is wanted, for each operand
    and entry; under no_grad the call goes on (to the next refusal, that of CPU tensors)."""
    group = SimpleNamespace(
        shapes=[(8, 64)], pair_bounds=[0, 256], row_bounds=[0, 8], qblock=64, qblock2=256,
        packed=torch.zeros(256, dtype=torch.uint8), absmax8=torch.zeros(8, dtype=torch.uint8),
        code=torch.zeros(256), absmax2=torch.zeros(1), offset2=torch.zeros(1),
        levels=torch.tensor(qgroup.NF4_LEVELS))
    t = {"x": torch.zeros(2, 64).half(), "bias": torch.zeros(8).half(),
         "lora_A": torch.zeros(4, 64), "lora_B": torch.zeros(8, 4), "out": torch.zeros(2, 8).half()}
    t[which].requires_grad_()

    def calls():
        extra = dict(bias=t["bias"], adapter=(t["lora_A"], t["lora_B"], 1.0))
        yield lambda: nf4_dequant.nf4_matvec(t["x"], group.packed, torch.zeros(8), 64, out=t["out"],
                                             **extra)
        yield lambda: qgroup.launch_matvec(t["x"], group.packed, group.absmax8, group.code,
                                           group.absmax2, group.offset2, group.levels, t["out"], 0, 8,
                                           64, 64, 256, **extra)
        if which != "out":
            yield lambda: qgroup.matvec(t["x"], group, 0, **extra)

    for call in calls():
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("first,last", [(-1, None), (-2, -1), (-1, 0), (0, 4), (3, None), (2, 1), (3, 3)])
def test_spans_outside_the_group_are_refused(first, last):
    """A negative index reaches a projection's shape but none of its bytes: the kernels would read
    past the group's buffers."""
    group = SimpleNamespace(
        shapes=[(8, 64), (16, 64), (8, 64)], pair_bounds=[0, 256, 768, 1024],
        row_bounds=[0, 8, 24, 32], qblock=64, qblock2=256, packed=torch.zeros(1024, dtype=torch.uint8),
        absmax8=torch.zeros(32, dtype=torch.uint8), code=torch.zeros(256), absmax2=torch.zeros(1),
        offset2=torch.zeros(1), levels=torch.tensor(qgroup.NF4_LEVELS))
    x = torch.zeros(2, 64).half()
    for call in (qgroup.matvec, qgroup.fused_linear):
        with pytest.raises(IndexError, match="of a group of 3"):
            call(x, group, first, last)
    packed, absmax8, row0, rows, cols = qgroup._span(group, 1, 3)
    assert (packed.numel(), absmax8.numel(), row0, rows, cols) == (768, 24, 8, 24, 64)
    assert qgroup._span(group, 1, 1)[3] == 0


@pytest.mark.parametrize("n_in,n_out", [(0, 8), (8, 0), (0, 0)])
def test_branch_of_no_columns_is_refused(n_in, n_out):
    with pytest.raises(ValueError, match="multiples of 8"):
        adapter.lora_branch(torch.zeros(4, n_in).half(), torch.zeros(4, n_out).half(),
                            torch.zeros(2, n_in), torch.zeros(n_out, 2), 1.0)


# ------------------------------------------------------------------------------------------
# memory that an output shares with the input
# ------------------------------------------------------------------------------------------
def test_outputs_in_the_inputs_memory_are_found():
    buffer = torch.randn(4, 160).half()
    x = buffer[:, :64]
    flat = torch.randn(4 * 64 + 8).half()
    square = flat[:256].view(4, 64)
    for rows, out, shared in (
            (square, square, True), (square, flat[8:264].view(4, 64), True),
            (square[:1], square[:1], True), (x, buffer[:, 32:96], True),
            (x, torch.empty(4, 64).half(), False), (square[:2], square[2:], False),
            (square[2:], square[:2], False), (square[:0], square[:0], False)):
        assert qgroup._share(rows.shape[0], rows.data_ptr(), rows.stride(0), 64, out.data_ptr(),
                             out.stride(0), 64) == shared


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 9, 32])
def test_product_written_over_its_input(rows):
    """A square projection in place, and beside its input in one buffer: the bits of a separate one."""
    g = torch.Generator().manual_seed(rows)
    size = 1536
    packed = torch.randint(0, 256, (size * size // 2,), generator=g, dtype=torch.uint8).cuda()
    absmax = (torch.rand(size * size // 64, generator=g) * 0.05).cuda()
    x = torch.randn(rows, size, generator=g).half().cuda()
    for extra in (None, ((torch.randn(8, size, generator=g) * 0.02).cuda(),
                         torch.randn(size, 8, generator=g).cuda(), 1.0)):
        want = nf4_dequant.nf4_matvec(x, packed, absmax, 64, adapter=extra)
        buffer = torch.zeros(rows, 2 * size, dtype=torch.float16, device="cuda")
        for a, b in ((0, 0), (0, 8), (0, size), (size, 0)):
            buffer[:, a:a + size] = x
            nf4_dequant.nf4_matvec(buffer[:, a:a + size], packed, absmax, 64,
                                   out=buffer[:, b:b + size], adapter=extra)
            assert torch.equal(buffer[:, b:b + size], want), (a, b)


@pytest.mark.parametrize("cols", [1, 2, 40])
def test_negated_views_are_written_out(cols):
    """The data of a lazily negated view (the imaginary part of a conjugate) has the other sign: what the
    kernels are given holds the view's values. One column is not copied for its stride."""
    real = torch.randn(30, cols, 2, generator=torch.Generator().manual_seed(1))
    view = torch.view_as_complex(real).conj().imag
    assert view.is_neg()
    rows, ld = adapter._rows(view, cols)
    assert not rows.is_neg() and ld >= cols and torch.equal(rows, -real[..., 1])


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [1, 40])
def test_dropout_of_a_negated_view(cols):
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")
    z = torch.randn(30, cols, dtype=torch.complex64, device="cuda")
    x = z.conj().imag
    assert x.is_neg()
    assert torch.equal(adapter.dropout(x, 0.3, seed), adapter.dropout((-z.imag).contiguous(), 0.3, seed))


@pytest.mark.gpu
def test_function_transforms_are_refused():
    """torch.func's transforms of the two training operators and of the few-row product end in an error,
    before any launch."""
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")
    x = torch.randn(3, 4, 64, device="cuda").half()
    base = torch.zeros(3, 4, 16, device="cuda").half()
    a, b = torch.randn(4, 64, device="cuda"), torch.randn(16, 4, device="cuda")
    packed = torch.zeros(16 * 32, dtype=torch.uint8, device="cuda")
    absmax = torch.ones(16, device="cuda")
    calls = (lambda v: adapter.dropout(v, 0.1, seed).float().sum(),
             lambda v: adapter.lora_branch(v, base[0], a, b, 1.0).float().sum(),
             lambda v: nf4_dequant.nf4_matvec(v, packed, absmax, 64).float().sum())
    for call in calls:
        with pytest.raises(RuntimeError):
            torch.func.grad(call)(x[0])
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(x)


# ------------------------------------------------------------------------------------------
# decoding
# ------------------------------------------------------------------------------------------
class _Counting(torch.nn.Module):
    """Predicts each token's successor; fails at the token 9."""

    def __init__(self):
        super().__init__()
        self.frozen, self.live = torch.nn.Dropout(0.5), torch.nn.Dropout(0.5)

    def forward(self, input_ids, past_key_values, use_cache, logits_to_keep):
        assert not (self.training or self.frozen.training or self.live.training)
        assert use_cache and qgroup._SERVING["rows"] == qgroup.MATVEC_MAX_ROWS
        last = input_ids[:, -1:]
        if (last == 9).any():
            raise RuntimeError("nine")
        logits = torch.nn.functional.one_hot(last + 1, 16).float()
        return SimpleNamespace(logits=logits, past_key_values=(past_key_values or 0) + 1)


def test_generate_leaves_every_module_in_its_own_mode():
    """A part in evaluation mode inside a model that trains stays there, also behind an error."""
    model = _Counting().train()
    model.frozen.eval()
    ids = torch.tensor([[1, 2], [4, 3]])
    assert qlora.generate(model, ids, 3).tolist() == [[1, 2, 3, 4, 5], [4, 3, 4, 5, 6]]
    assert model.training and model.live.training and not model.frozen.training
    with pytest.raises(RuntimeError, match="nine"):
        qlora.generate(model, ids, 9)
    assert model.training and model.live.training and not model.frozen.training
    assert qgroup._SERVING["rows"] == 0
    model.eval()
    model.live.train()
    assert torch.equal(qlora.generate(model, ids, 0), ids)
    assert not model.training and model.live.training


# ------------------------------------------------------------------------------------------
# bookkeeping
# ------------------------------------------------------------------------------------------
def test_every_component_is_one_that_some_call_reports():
    """The components of state.py are those that a call site records a failure of."""
    package = os.path.dirname(state.__file__)
    reported = set()
    for name in os.listdir(package):
        if name.endswith(".py"):
            with open(os.path.join(package, name)) as f:
                reported |= set(re.findall(r'fallback\("(\w+)"', f.read()))
    assert reported == set(state.COMPONENTS)


@pytest.mark.parametrize("short", [True, False])
def test_stream_and_device_without_the_short_ways(monkeypatch, short):
    """A PyTorch without the private calls is asked through the public ones."""
    x = SimpleNamespace(get_device=lambda: 3)
    entered = []
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: SimpleNamespace(cuda_stream=100 + d))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "device", lambda d: entered.append(d))
    monkeypatch.setattr(_lib, "_CURRENT_STREAM", (lambda d: 200 + d) if short else None)
    monkeypatch.setattr(_lib, "_CURRENT_DEVICE", (lambda: 5) if short else None)
    assert _lib.raw_stream(x) == (203 if short else 103)
    _lib.device_of(x)
    assert entered == ([3] if short else [])
