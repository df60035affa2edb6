"""The training form of a LoRA adapter, with counter-based dropout inside it.

  dropout(x, p, seed)                               dropout whose mask is never stored
  lora_branch(x, base, lora_A, lora_B, scaling, p, seed)
                                                    base + scaling * (dropout(x) A^T) B^T
  draw_seed(device)                                 the seed of one call, from torch's generator

Both are autograd functions over the kernels of csrc/adapter.cu. The mask of a call is a function of
its seed and of the element's place in row-major order (Philox4x32 with 7 rounds; element e of `x` is
kept when the low 15 bits of half e % 8 of counter e / 8 reach round(p * 32768)), so the backward
pass makes it again instead of reading it: no dropped copy of the input and no mask are kept. With
the rank rounded up to R = 16, 32 or 64, the branch saves its input, the seed, the rank-wide product
(max(128, 4 R) bytes a row and R / 32 for its scales) and the adapter as it was, in the kernels'
parts (4 R bytes per output and max(128, 4 R) per input column). The probability is thereby rounded
to a multiple of 1 / 32768; the factor 32768 / (32768 - drop) is that of the rounded one, which
keeps the expectation.

The seed is a one-element int64 tensor on the device. `draw_seed` fills it from torch's own CUDA
generator: torch.manual_seed makes a run repeatable, a captured graph draws a new seed on every
replay, and gradient checkpointing, which restores the generator, recomputes the same mask.

The reference's adapter node (solution/lora.py:151-231) keeps the dropout's generator state and
replays it in the backward; its products run in fp16. Here sums are fp32 and each fp16 result is
rounded once. There is no CPU path, a failing call raises (no component is turned off by it), and
like GroupLinear neither function takes part in torch.func's transforms, which refuse it.
"""

import functools
import math

import torch

from . import _lib
from .engaged import RAN

MAX_RANK = 64
DROP_ALL = 32768
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # TALM_DTYPE_*


def draw_seed(device):
    """A seed for one call: int64 [1] on `device`, drawn from torch's CUDA generator."""
    return torch.empty(1, dtype=torch.int64, device=device).random_()


def drop_threshold(p):
    """round(p * 32768): the number of the 32768 values of a draw that drop an element."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability has to be between 0 and 1, got {p}")
    return math.floor(p * DROP_ALL + 0.5)


def _check_seed(seed, x):
    if (not torch.is_tensor(seed) or seed.dtype is not torch.int64 or seed.numel() != 1
            or seed.get_device() != x.get_device()):
        raise ValueError("seed must be an int64 tensor of one element on the input's device")


def _rows(t, cols):
    """`t` as [rows, cols] rows of unit stride that do not overlap (a view where its strides
    allow it, else a copy), and their stride. A lazily negated view (the imaginary part of a conjugate)
    is written out."""
    if t.is_neg():
        t = t.resolve_neg()
    if t.is_contiguous():
        return t, cols
    t = t.reshape(-1, cols)
    ld, unit = t.stride()
    if t.shape[0] == 1:
        ld = cols
    if (unit != 1 and cols > 1) or ld < cols:
        t, ld = t.contiguous(), cols
    return t, ld


def _rows16(t, cols):
    """`_rows` on 16-byte boundaries, as the branch's kernels read them."""
    t, ld = _rows(t, cols)
    if t.data_ptr() % 16 or ld % 8:
        t, ld = t.clone(memory_format=torch.contiguous_format), cols
    return t, ld


def _run_dropout(x, seed, drop):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    n = x.numel()
    if n:
        cols = x.shape[-1] if x.dim() else 1
        rows, ld = _rows(x, cols)
        with _lib.device_of(x):
            _lib.check(_lib.load().talm_dropout(
                rows.data_ptr(), ld, n // cols, cols, _DTYPES[x.dtype], seed.data_ptr(), drop,
                y.data_ptr(), _lib.raw_stream(x)), "talm_dropout")
        RAN["dropout"] += 1
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, seed, drop):
        ctx.drop = drop
        ctx.save_for_backward(seed)
        return _run_dropout(x, seed, drop)

    @staticmethod
    def backward(ctx, grad):
        (seed,) = ctx.saved_tensors
        # the same map; through the node again only where its own gradient is wanted
        run = _Dropout.apply if torch.is_grad_enabled() else _run_dropout
        return run(grad, seed, ctx.drop), None, None


def dropout(x, p, seed):
    """x * mask * 32768 / (32768 - drop), drop = round(p * 32768), the mask a function of `seed`
    and the element's index. x: fp16, bf16 or fp32 of any shape and strides on a CUDA device; a
    dropped element gives 0 whatever x holds. Differentiable (twice as well)."""
    if x.dtype not in _DTYPES:
        raise TypeError(f"dropout takes fp16, bf16 or fp32, got {x.dtype}")
    drop = drop_threshold(p)
    _lib.ptr(x)
    _check_seed(seed, x)
    return _Dropout.apply(x, seed, drop)


def branch_takes(x, base, rank):
    """Whether `lora_branch` takes this call: fp16 on one CUDA device, widths of multiples of 8,
    a rank of at most MAX_RANK."""
    return (x.is_cuda and x.dtype == torch.float16 and base.dtype == torch.float16
            and x.shape[-1] % 8 == 0 and base.shape[-1] % 8 == 0 and 1 <= rank <= MAX_RANK)


@functools.lru_cache(maxsize=256)
def _sizes(n_rows, n_in, n_out, rank):
    saved, forward, backward = _lib._SZ(0), _lib._SZ(0), _lib._SZ(0)
    _lib.check(_lib.load().talm_lora_sizes(n_rows, n_in, n_out, rank, saved, forward, backward),
               "talm_lora_sizes")
    return saved.value, forward.value, backward.value


def _bytes(n, x):
    return torch.empty(n, dtype=torch.uint8, device=x.device)


class _LoraBranch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, base, lora_a, lora_b, scaling, seed, drop, want_grad):
        n_in, n_out, rank = x.shape[-1], base.shape[-1], lora_a.shape[0]
        n_rows = base.numel() // n_out
        a, b = lora_a.contiguous(), lora_b.contiguous()
        xr, ld_x = _rows16(x, n_in)
        br, ld_b = _rows16(base, n_out)
        saved_bytes, work_bytes, ctx.work_bytes = _sizes(n_rows, n_in, n_out, rank)
        y = torch.empty(base.shape, dtype=torch.float16, device=x.device)
        saved = _bytes(saved_bytes, x) if want_grad else None
        work = _bytes(work_bytes, x)
        with _lib.device_of(x):
            _lib.check(_lib.load().talm_lora_forward(
                xr.data_ptr(), ld_x, br.data_ptr(), ld_b, a.data_ptr(), b.data_ptr(), n_rows,
                n_in, n_out, rank, scaling, None if seed is None else seed.data_ptr(), drop,
                y.data_ptr(), None if saved is None else saved.data_ptr(), saved_bytes,
                work.data_ptr(), work_bytes, _lib.raw_stream(x)), "talm_lora_forward")
        if want_grad:  # `saved` holds the adapter as it is now, in the kernels' parts
            ctx.scaling, ctx.drop, ctx.rank = scaling, drop, rank
            ctx.save_for_backward(x, seed, saved)
        RAN["lora"] += 1
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        need_x, need_base, need_a, need_b = ctx.needs_input_grad[:4]
        dx = da = db = None
        if need_x or need_a or need_b:
            x, seed, saved = ctx.saved_tensors
            n_in, n_out, rank = x.shape[-1], grad.shape[-1], ctx.rank
            device = x.device
            if need_x:
                dx = torch.empty(x.shape, dtype=torch.float16, device=device)
            if need_a:
                da = torch.empty((rank, n_in), dtype=torch.float32, device=device)
            if need_b:
                db = torch.empty((n_out, rank), dtype=torch.float32, device=device)
            xr, ld_x = _rows16(x, n_in)
            gr, ld_g = _rows16(grad, n_out)
            work = _bytes(ctx.work_bytes, x)
            with _lib.device_of(x):
                _lib.check(_lib.load().talm_lora_backward(
                    gr.data_ptr(), ld_g, xr.data_ptr(), ld_x, saved.data_ptr(), saved.numel(),
                    grad.numel() // n_out, n_in, n_out, rank, ctx.scaling,
                    None if seed is None else seed.data_ptr(), ctx.drop,
                    dx.data_ptr() if need_x else None, da.data_ptr() if need_a else None,
                    db.data_ptr() if need_b else None, work.data_ptr(), ctx.work_bytes,
                    _lib.raw_stream(x)), "talm_lora_backward")
        return dx, grad if need_base else None, da, db, None, None, None, None


def lora_branch(x, base, lora_A, lora_B, scaling, p=0.0, seed=None):
    """base + scaling * (dropout(x) A^T) B^T, rounded to fp16 once, with gradients for x, base, A
    and B. x [..., in] and base [..., out]: fp16 with the same leading sizes; lora_A [r, in] and
    lora_B [out, r]: fp32, r in 1..64; `in` and `out` multiples of 8. p > 0 takes a `seed`
    (`draw_seed`); the mask is that of `dropout(x, p, seed)`."""
    n_in, n_out = x.shape[-1], base.shape[-1]
    if x.dtype is not torch.float16 or base.dtype is not torch.float16:
        raise TypeError(f"lora_branch takes fp16 x and base, got {x.dtype} and {base.dtype}")
    if lora_A.dtype is not torch.float32 or lora_B.dtype is not torch.float32:
        raise TypeError("lora_A and lora_B must be fp32")
    if x.shape[:-1] != base.shape[:-1]:
        raise ValueError(f"x {tuple(x.shape)} and base {tuple(base.shape)} differ in their rows")
    rank = lora_A.shape[0]
    if lora_A.shape != (rank, n_in) or lora_B.shape != (n_out, rank):
        raise ValueError(f"adapter {tuple(lora_A.shape)}, {tuple(lora_B.shape)} does not map "
                         f"{n_in} to {n_out}")
    if not 1 <= rank <= MAX_RANK or n_in < 8 or n_out < 8 or n_in % 8 or n_out % 8:
        raise ValueError(f"lora_branch needs a rank of 1..{MAX_RANK} and widths of multiples of "
                         f"8, got rank {rank}, {n_in} -> {n_out}")
    drop = drop_threshold(p)
    device = x.get_device()
    if device < 0:
        raise RuntimeError("talm_b200 kernels run on CUDA tensors only (no CPU path)")
    if not base.get_device() == lora_A.get_device() == lora_B.get_device() == device:
        raise ValueError("x, base and the adapter must be on one device")
    if drop == 0:
        seed = None
    else:
        if seed is None:
            raise ValueError("dropout needs a seed (adapter.draw_seed)")
        _check_seed(seed, x)
    want_grad = torch.is_grad_enabled() and (x.requires_grad or lora_A.requires_grad
                                             or lora_B.requires_grad)
    return _LoraBranch.apply(x, base, lora_A, lora_B, float(scaling), seed, drop, want_grad)
